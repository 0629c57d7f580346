"""Attention over a cache in 4 bits on the GPU where the precision of its parts shows (helpers: test_kv4_gpu.py)."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import l2domain_b200 as L  # noqa: E402
from test_decode_ops_gpu import TORCH, U, close, gen, gpu  # noqa: E402,F401
from test_kv4_gpu import Pages4, stand_for  # noqa: E402


@pytest.mark.parametrize("dt", [L.F16, L.F32])
@pytest.mark.parametrize("group,D", [(32, 32), (32, 100), (64, 64), (64, 128), (128, 128), (128, 256)])
@pytest.mark.parametrize("G", [1, 8, 12])
def test_weights_keep_what_fp32_holds(dt, group, D, G):
    """Two keys whose values are each other's negatives, with nearly equal weights: an output is the difference of the weights,
    v times.  Per weight, in units u = 2^-24: a score is one product, scaled twice, and log2(e) and the scale are rounded, 5 u of a
    score below 1; less the largest, a rounding; exp2, 4 u; times the value's scale and a power of two, 1 u: 11 u of the weight.  The
    products: three parts, each instruction cuts three operands off at the last place of the largest, 2 u each: 18 u.  Of both: 40 u
    of sum w |v|; dividing by the sum of weights, 8 u of the output alone."""
    B, heads = 64, 2
    P = Pages4(dt, B, 1, 16, heads, D, group, seed=D + G)
    g = gen(D)
    k, v = torch.zeros(P.num_pages, 16, heads, D, device="cuda"), torch.zeros(P.num_pages, 16, heads, D, device="cuda")
    k[:, 0, :, 0] = 1.0
    v[:, 0] = torch.empty(P.num_pages, heads, D, device="cuda").uniform_(0.0, 3.0, generator=g)
    v[:, 1] = -v[:, 0]
    P.k, P.v = (stand_for(*P.fill(i, x), group) for i, x in enumerate((k, v)))
    q = torch.zeros(B, heads * G, D, dtype=TORCH[dt], device="cuda")
    q[..., 0] = torch.empty(B, heads * G, device="cuda").uniform_(-0.06, 0.06, generator=g).to(TORCH[dt])
    out = torch.full_like(q, math.nan)
    plan = L.PagedAttention(P.cache(), P.table, B, 1, heads * G, scale=1.0)
    plan.decode(q, out, torch.full((B,), 2, dtype=torch.int32, device="cuda"), B)
    torch.cuda.synchronize()
    at = P.table[:, 0].long()
    k, v = P.k[at, :2].repeat_interleave(G, 2), P.v[at, :2].repeat_interleave(G, 2)
    w = torch.softmax(torch.einsum("bhd,bnhd->bnh", q.double(), k), 1)
    want = torch.einsum("bnh,bnhd->bhd", w, v)
    close(out, want, 40 * U * torch.einsum("bnh,bnhd->bhd", w, v.abs()) + 8 * U * want.abs(), dt)
