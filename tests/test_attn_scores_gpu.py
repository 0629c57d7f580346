"""Attention with other scores (caps, biases by distance, starts of documents) on the GPU against its definition in 64
bits, over caches of 32, 16 and 4 bits.  Tolerances as in test_kv4_gpu.py; caches of 16 bits leave 2^-16 of a weight (bf16) or
2^-20 of it and 2^-40 of the largest (fp16, `least`), of 32 bits nothing."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import l2domain_b200 as L  # noqa: E402
from test_decode_ops_gpu import TORCH, Pages, gen, gpu, normal  # noqa: E402,F401
from test_kv4_gpu import Pages4, check  # noqa: E402

PARTS = {L.F32: 0.0, L.F16: 2.0 ** -20, L.BF16: 2.0 ** -16}


def kept(parts, dt):
    """What check() needs to know of a cache: nothing where it is in 4 bits (parts is None)."""
    return dict(parts=parts, least=2.0 ** -40 if parts is not None and dt == L.F16 else 2.0 ** -104)


def pages(bits, dt, seqs, width, page, heads, D, seed=0):
    if bits == 4:
        return Pages4(dt, seqs, width, page, heads, D, 32, seed=seed), None
    return Pages(dt, seqs, width, page, heads, D, seed=seed), PARTS[dt]


def some_slopes(heads, seed):
    return torch.empty(heads, device="cuda").uniform_(-0.2, 0.5, generator=gen(seed))


@pytest.mark.parametrize("bits", [0, 4])
@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("heads,G,D", [(1, 1, 64), (3, 2, 128), (2, 8, 80), (1, 12, 128), (2, 16, 64), (1, 33, 192), (2, 4, 256), (1, 16, 256), (4, 1, 160), (1, 5, 96), (1, 16, 96)])
def test_caps_and_slopes(bits, dt, heads, G, D):
    P, parts = pages(bits, dt, 5, 20, 16, heads, D, seed=G)
    lens = [300, 0, 1, 17, 255]
    slopes = some_slopes(heads * G, D)
    check(P, lens, heads * G, dt, cap=3.0, **kept(parts, dt))
    check(P, lens, heads * G, dt, slopes=slopes, **kept(parts, dt))
    check(P, lens, heads * G, dt, scale=-0.3, cap=30.0, slopes=slopes, starts=[100, 0, 1, 3, 254], window=150, **kept(parts, dt))


@pytest.mark.parametrize("bits", [0, 4])
@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_long_sequences_cut_between_blocks(bits, dt):
    lens = [9000, 3, 0, 2048, 5001]
    P, parts = pages(bits, dt, 5, 282, 32, 2, 64, seed=3)
    slopes = L.distance_slopes(8, device="cuda")
    for kw in (dict(cap=2.0), dict(slopes=slopes), dict(cap=20.0, slopes=slopes, starts=[1, 0, 9, 2000, 4000])):
        first = check(P, lens, 8, dt, **kept(parts, dt), **kw)
        again = check(P, lens, 8, dt, **kept(parts, dt), **kw)
        assert all(torch.equal(a[:-1], b[:-1]) for a, b in zip(first, again))


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("layout", ["heads first", "odd"])
@pytest.mark.parametrize("page", [1, 7])
def test_layouts_and_odd_pages(dt, layout, page):
    P = Pages(dt, 3, -(-230 // page), page, 2, 64, layout, seed=page)
    check(P, [230, 65, 7], 8, dt, cap=5.0, slopes=some_slopes(8, 1), starts=[77, 0, 2], **kept(PARTS[dt], dt))


@pytest.mark.parametrize("bits", [0, 4])
@pytest.mark.parametrize("dt", [L.F32, L.BF16])
def test_starts_without_other_scores(bits, dt):
    """Documents that begin at the front, inside a tile, at its end, at the last position, and behind it: rows of none."""
    P, parts = pages(bits, dt, 8, 40, 16, 2, 64, seed=4)
    lens = [640, 640, 640, 640, 640, 100, 0, 5]
    starts = [0, 1, 127, 128, 639, 100, 0, 2 ** 31 - 1]
    out, lse = check(P, lens, 4, dt, starts=starts, **kept(parts, dt))
    assert (out[5:8] == 0).all() and (lse[5:8] == -math.inf).all()
    # Pages before a document's start may have been given back.
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for b, (n, s) in enumerate(zip(lens, starts)):
        P.table[b, : min(s, n) // 16] = -1
        P.table[b, -(-n // 16):] = -1
    plan = L.PagedAttention(P.cache(), P.table, 8, 40, 4, status=status)
    again, _ = check(P, lens, 4, dt, starts=starts, **kept(parts, dt), plan=plan)
    assert status.item() == 0 and torch.equal(out[:8], again[:8])


@pytest.mark.parametrize("bits", [0, 4])
@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_caps_of_large_scores_and_steep_slopes(bits, dt):
    """Scores of thousands under a cap are all but the cap; a bias that falls by 40 a position leaves the last key."""
    P, parts = pages(bits, dt, 2, 20, 16, 2, 64, seed=5)
    q = normal(gen(2), dt, 2, 4, 64) * 50
    check(P, [300, 31], 4, dt, cap=8.0, scale=0.5, q=q, **kept(parts, dt))
    slopes = torch.tensor([40.0, 0.0, 1e-6, 100.0], device="cuda")
    out, _ = check(P, [300, 31], 4, dt, slopes=slopes, **kept(parts, dt))
    last = P.rows(0, 299, 300)[1][0, 0].double()
    assert (out[0, 0].double() - last).abs().max() <= 2.0 ** -8 * last.abs().max()


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
def test_infinite_scores_under_a_cap(dt):
    """A score of -inf is one of -cap, as its tanh is -1; a NaN stays one."""
    P = Pages(dt, 2, 6, 16, 1, 64, seed=4)
    q = torch.ones(2, 1, 64, dtype=TORCH[dt], device="cuda")
    P.k[int(P.table[0, 2]), 8] = -math.inf
    P.k[int(P.table[1, 0]), 5] = math.nan
    out, lse = torch.empty_like(q), torch.empty(2, 1, device="cuda")
    L.PagedAttention(P.cache(), P.table, 2, 6, 1, cap=2.0).decode(q, out, torch.tensor([90, 90], dtype=torch.int32, device="cuda"), 2, lse=lse)
    k, v = (t[:, 0].double() for t in P.rows(0, 0, 90))
    s = 2.0 * torch.tanh((k @ q[0, 0].double()) / 8.0 / 2.0)
    assert s[40] == -2.0
    assert (out[0, 0].double() - torch.softmax(s, 0) @ v).abs().max() < (1e-5 if dt == L.F32 else 2e-2)
    assert abs(lse[0, 0].item() - torch.logsumexp(s, 0).item()) < 1e-5
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()


def test_plain_plans_are_as_before():
    """No cap and no slopes: the bits of a plan made without scores; starts of 0 change nothing."""
    P = Pages(L.BF16, 3, 40, 16, 2, 128, seed=6)
    q, lens = normal(gen(1), L.BF16, 3, 8, 128), torch.tensor([640, 77, 0], dtype=torch.int32, device="cuda")
    import ctypes as C
    plan = C.c_void_p(0)
    cd, ad = P.cache().desc(P.table, 3, 40), L.AttnDesc(heads_q=8)
    L.check(L.lib().l2d_attn_plan_create(C.byref(cd), C.byref(ad), C.byref(plan)))
    a, b = torch.empty_like(q), torch.empty_like(q)
    L.check(L.lib().l2d_attn_decode(plan, q.data_ptr(), a.data_ptr(), None, lens.data_ptr(), 3, None))
    L.PagedAttention(P.cache(), P.table, 3, 40, 8).decode(q, b, lens, 3, starts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    L.check(L.lib().l2d_attn_plan_destroy(plan))
    assert torch.equal(a, b)


def test_slopes_may_change_between_calls():
    """A plan reads its slopes when it runs, in the order of the stream."""
    P = Pages(L.F32, 1, 10, 16, 1, 64, seed=7)
    slopes = torch.zeros(2, device="cuda")
    plan = L.PagedAttention(P.cache(), P.table, 1, 10, 2, slopes=slopes)
    check(P, [150], 2, L.F32, slopes=slopes, plan=plan, parts=0.0)
    slopes.copy_(torch.tensor([0.3, -0.1]))
    check(P, [150], 2, L.F32, slopes=slopes, plan=plan, parts=0.0)
