"""Packing of 4-bit weights (CPU), and the decoding layer built from the operators against 64-bit arithmetic (GPU)."""
import math

import pytest

torch = pytest.importorskip("torch")

import l2domain_b200 as L  # noqa: E402
from l2domain_b200.decode import DecodeAttention, pack_q4  # noqa: E402


def unpack(packed, scales, zeros, N, group):
    col = torch.arange(N, device=packed.device)
    q = ((packed[:, col // 2].long() >> (4 * (col % 2))) & 15).double()
    z = zeros[:, col // group].double() if zeros is not None else 8.0
    return (q - z) * scales[:, col // group].double()


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("M,N,group", [(5, 256, 32), (3, 100, 64), (2, 131, 128), (1, 7, 32)])
def test_packing_is_within_half_a_step(M, N, group, zero_points):
    g = torch.Generator().manual_seed(N)
    w = torch.randn(M, N, generator=g)
    if zero_points:
        w = w.abs() + 0.5  # one-sided ranges
    packed, scales, zeros = pack_q4(w, group, zero_points, L.F32)
    assert packed.shape[1] % 16 == 0 and scales.shape[1] % 8 == 0 and (zeros is not None) == zero_points
    step = scales[:, torch.arange(N) // group].double()
    # half a step, or up to a whole one where zero point and value are both rounded
    slack = (1.0 if zero_points else 0.5) * step * (1 + 1e-6) + 1e-12
    assert ((unpack(packed, scales, zeros, N, group) - w.double()).abs() <= slack).all()


def test_packing_of_zeros():
    packed, scales, zeros = pack_q4(torch.zeros(2, 64), 32)
    assert (unpack(packed, scales, zeros, 64, 32) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads,kv_heads,head_dim,hidden", [(3, 4, 2, 64, 256), (1, 8, 1, 128, 384)])
def test_layer_follows_its_definition(batch, heads, kv_heads, head_dim, hidden):
    """Forty steps from an empty cache: each stage against 64-bit arithmetic on the bf16 inputs it was given, so an
    error is one rounding to bf16 (2^-8 relative to the row's largest terms) and not a chain of them."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    g = torch.Generator(device="cuda").manual_seed(heads)
    row = (heads + 2 * kv_heads) * head_dim

    def normal(*shape, scale=1.0):
        return (torch.empty(shape, device="cuda").normal_(generator=g) * scale).to(torch.bfloat16)

    w_qkv, w_out = normal(row, hidden, scale=hidden ** -0.5), normal(hidden, heads * head_dim, scale=0.1)
    layer = DecodeAttention(w_qkv, w_out, heads, kv_heads, head_dim, batch, 64)
    exact_qkv, exact_out = (unpack(*pack_q4(w, 128, dtype_s=L.BF16), w.shape[1], 128) for w in (w_qkv, w_out))
    keys, values = [], []
    out = torch.empty(batch, hidden, dtype=torch.bfloat16, device="cuda")
    freq = 10000.0 ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device="cuda") / head_dim)
    half = head_dim // 2

    def near(got, want):
        assert (got.double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()

    for t in range(40):
        x = normal(batch, hidden)
        pos = torch.full((batch,), t, dtype=torch.int32, device="cuda")
        layer.step(x, pos, pos + 1, out)
        torch.cuda.synchronize()
        plain = (x.double() @ exact_qkv.t()).view(batch, -1, head_dim)
        angle = t * freq
        a, b = plain[..., :half], plain[..., half:]
        turned = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)
        got = layer.qkv.view(batch, -1, head_dim)
        near(got[:, :heads], turned[:, :heads])
        page, slot = layer.table[:, t // 16].long(), t % 16
        near(layer.k[page, slot], turned[:, heads: heads + kv_heads])
        near(layer.v[page, slot], plain[:, heads + kv_heads:])
        keys.append(layer.k[page, slot].double())
        values.append(layer.v[page, slot].double())
        k, v = (torch.stack(z, 1).repeat_interleave(heads // kv_heads, 2) for z in (keys, values))
        w = torch.softmax(torch.einsum("bhd,bnhd->bhn", got[:, :heads].double(), k) / math.sqrt(head_dim), -1)
        near(layer.mixed.view(batch, heads, head_dim), torch.einsum("bhn,bnhd->bhd", w, v))
        near(out, layer.mixed.double() @ exact_out.t())
    assert layer.status.item() == 0
