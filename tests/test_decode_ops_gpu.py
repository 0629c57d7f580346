"""The decoding operators on the GPU against their definitions in 64 bits.

Tolerances, per element, from rounding alone (u = 2^-24; the kernels may sum in any order, and a matrix
instruction may truncate where it adds, which costs twice a rounding):

* q4: the products (q - z) x are exact.  A sum of n terms in partial sums of at most 160 + n / 32 additions
  in a row, each off by 2u of what it holds, is off by 2u (160 + n / 32) S with S the sum of the terms'
  absolute values; the output's own rounding comes on top.
* attention: a score is off by d = 2u (D + 8) |scale| sum|q k|, so a weight by a factor of at most 1 + 2 d
  and some 2^-20 for exp; in 16-bit caches a weight may be rounded once to the cache's type (u16).  Sums add
  2u (160 + n / 16).  All of it is relative to sum w |v|.
* append: two products and a sum in fp32, 4u (|a| + |b|), then one rounding; copied elements are equal.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import l2domain_b200 as L  # noqa: E402

TORCH = {L.F32: torch.float32, L.F16: torch.float16, L.BF16: torch.bfloat16}
U = 2.0 ** -24
U_OUT = {L.F32: 2.0 ** -24, L.F16: 2.0 ** -11, L.BF16: 2.0 ** -8}  # half a unit in the last place, relative (bf16: 8 bits)
TINY = {L.F32: 2.0 ** -126, L.F16: 2.0 ** -24, L.BF16: 2.0 ** -126}


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, dt, *shape):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=g).to(TORCH[dt])


def offset_view(t, elements):
    """A copy of t whose first element is `elements` past an aligned address."""
    buf = torch.zeros(t.numel() + elements, dtype=t.dtype, device=t.device)
    view = buf[elements:].view(t.shape)
    view.copy_(t)
    return view


def close(got, want, slack, dt):
    """|got - want| <= slack + one rounding of the result to dt."""
    tol = slack + U_OUT[dt] * (want.abs() + slack) + TINY[dt]
    err = (got.double() - want).abs()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the tolerance"


# ------------------------------------------------------------------------------------------------
# 4-bit products
# ------------------------------------------------------------------------------------------------

def q4_case(M, N, group, dt, vectors=1, zeros=False, dt_s=L.F16, pad_w=0, pad_s=0, seed=0):
    g = gen(seed)
    groups = -(-N // group)
    w = torch.randint(0, 256, (M, (N + 1) // 2 + pad_w), dtype=torch.uint8, device="cuda", generator=g)
    s = torch.empty(M, groups + pad_s, device="cuda").uniform_(-0.02, 0.02, generator=g).to(TORCH[dt_s])
    z = torch.randint(0, 256, (M, groups + pad_s), dtype=torch.uint8, device="cuda", generator=g) if zeros else None
    return w, s, z, normal(g, dt, vectors, N)


def q4_exact(w, s, z, x, N, group):
    """(y, S): the sums and the sums of absolute values, in 64 bits."""
    col = torch.arange(N, device="cuda")
    q = ((w[:, col // 2].long() >> (4 * (col % 2))) & 15).double()
    zero = (z[:, col // group].long() & 15).double() if z is not None else 8.0
    full = (q - zero) * s[:, col // group].double()
    return x.double() @ full.t(), x.double().abs() @ full.abs().t()


def q4_check(w, s, z, x, N, group, dt, dt_y=None, dt_s=L.F16, stream=None):
    M, vectors = w.shape[0], x.shape[0]
    dt_y = dt if dt_y is None else dt_y
    y = torch.full((vectors, M + 3), math.nan, dtype=TORCH[dt_y], device="cuda")
    m = L.Q4Matrix(w, s, M, N, group, zeros=z, dtype_x=dt, dtype_y=dt_y, dtype_s=dt_s, ldw=w.stride(0), lds=s.stride(0))
    m.gemv(x, y, vectors=vectors, stride_x=x.stride(0), stride_y=M + 3, stream=stream)
    torch.cuda.synchronize()
    want, total = q4_exact(w, s, z, x, N, group)
    close(y[:, :M], want, 2 * U * (160 + N / 32) * total, dt_y)
    assert torch.isnan(y[:, M:]).all()  # nothing past a vector's rows
    return y[:, :M].clone()


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("group", [32, 64, 128, 384])
@pytest.mark.parametrize("zeros", [False, True])
def test_q4_types_and_groups(dt, group, zeros):
    for vectors in (1, 3):
        q4_check(*q4_case(77, 1152, group, dt, vectors, zeros, seed=group), 1152, group, dt)


@pytest.mark.parametrize("M,N", [(1, 1), (1, 2), (3, 31), (5, 33), (16, 127), (17, 129), (33, 1000), (250, 5003), (40, 20481), (2, 70000)])
def test_q4_odd_sizes(M, N):
    for dt in (L.BF16, L.F32):
        q4_check(*q4_case(M, N, 64, dt, 2, True, seed=N), N, 64, dt)


@pytest.mark.parametrize("vectors", [1, 2, 4, 5, 7, 8, 9, 16, 17, 33])
@pytest.mark.parametrize("dt,group", [(L.BF16, 128), (L.F16, 32), (L.F32, 64), (L.F32, 32)])
def test_q4_vectors(vectors, dt, group):
    q4_check(*q4_case(100, 640, group, dt, vectors, vectors % 2 == 1, seed=vectors), 640, group, dt)


@pytest.mark.parametrize("dt_y", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("dt_s", [L.F32, L.F16, L.BF16])
def test_q4_output_and_scale_types(dt_y, dt_s):
    q4_check(*q4_case(65, 512, 128, L.F16, 2, False, dt_s, seed=3), 512, 128, L.F16, dt_y, dt_s)


@pytest.mark.parametrize("pad_w", [1, 2, 4, 8, 16, 31])
def test_q4_strides_and_alignment(pad_w):
    w, s, z, x = q4_case(70, 1000, 32, L.BF16, 3, True, pad_w=pad_w, pad_s=pad_w, seed=pad_w)
    first = q4_check(w, s, z, x, 1000, 32, L.BF16)
    shifted = offset_view(w, pad_w), offset_view(s, 1), offset_view(z, 1), offset_view(x, 1)
    assert torch.equal(first, q4_check(*shifted, 1000, 32, L.BF16))  # alignment does not change the bits


def test_q4_many_rows_and_long_rows():
    q4_check(*q4_case(20000, 256, 128, L.F16, 1, seed=1), 256, 128, L.F16)
    q4_check(*q4_case(48, 60000, 128, L.F16, 8, True, seed=2), 60000, 128, L.F16)
    q4_check(*q4_case(300, 16384, 32, L.F32, 4, True, seed=2), 16384, 32, L.F32)


def test_q4_extreme_activations():
    """Tiny and huge activations keep their bits; an infinity or a NaN reaches its own vector only."""
    w, s, z, x = q4_case(64, 512, 128, L.F32, 5, True, seed=4)
    x[0] *= 2.0 ** 100
    x[1] *= 2.0 ** -100
    x[2] = x[2] * torch.exp2(torch.randint(-40, 40, x[2].shape, device="cuda", generator=gen(5)).float())
    q4_check(w, s, z, x, 512, 128, L.F32)
    good = q4_check(w, s, z, x, 512, 128, L.F32)
    w[:, 16 // 2] = 0x3F  # q - z at columns 16, 17 is 15 - z and 3 - z
    z.fill_(4)
    good = q4_check(w, s, z, x, 512, 128, L.F32)
    x[1, 16] = math.inf
    x[3, 17] = math.nan
    y = torch.empty(5, 64, device="cuda")
    L.Q4Matrix(w, s, 64, 512, 128, zeros=z, dtype_x=L.F32).gemv(x, y, vectors=5)
    assert torch.isinf(y[1]).all() and torch.equal(torch.sign(y[1]), torch.sign(s[:, 0].float()))
    assert torch.isnan(y[3]).all()
    for b in (0, 2, 4):
        assert torch.equal(y[b], good[b])


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_q4_no_columns_gives_zeros(dt):
    y = torch.full((2, 9), math.nan, dtype=TORCH[dt], device="cuda")
    L.Q4Matrix(None, None, 9, 0, 128, dtype_x=dt).gemv(None, y, vectors=2)
    assert torch.equal(y, torch.zeros_like(y))


def test_q4_vector_alone_equals_vector_in_company():
    w, s, z, x = q4_case(200, 2048, 64, L.BF16, 8, True, seed=6)
    both = q4_check(w, s, z, x, 2048, 64, L.BF16)
    again = q4_check(w, s, z, x, 2048, 64, L.BF16)
    assert torch.equal(both, again)


@pytest.mark.parametrize("vectors", [1, 3, 9])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dt,dt_y", [(L.F32, L.F32), (L.BF16, L.F32)])
def test_q4_one_sided_activations_do_not_cancel(vectors, group, dt, dt_y):
    """Activations around 100: the sums of q x and of z x are hundreds of times the result.  An fp32 result is held to
    the rounding of sums of (q - z) x themselves: at most 8 products in a row in a matrix instruction's sum, each off
    by 2u of what it holds, and 2048 / 128 + 16 additions of groups' sums."""
    w, s, z, x = q4_case(150, 2048, group, dt, vectors, True, seed=7)
    x = (x.float() + 100).to(TORCH[dt])
    y = torch.empty(vectors, 150, dtype=TORCH[dt_y], device="cuda")
    L.Q4Matrix(w, s, 150, 2048, group, zeros=z, dtype_x=dt, dtype_y=dt_y, ldw=w.stride(0), lds=s.stride(0)).gemv(x, y, vectors=vectors)
    want, total = q4_exact(w, s, z, x, 2048, group)
    close(y, want, 2 * U * (8 + 2048 / 128 + 16) * total, dt_y)


@pytest.mark.parametrize("N,group", [(4096, 128), (2048, 64), (1536, 32), (4096, 512), (4224, 384), (11008, 128), (5120, 256)])
@pytest.mark.parametrize("vectors", [1, 2, 6])
def test_q4_whole_steps_and_remainders(N, group, vectors):
    """Rows of whole 512-column steps and of steps and a rest, with scales read in words and by twos."""
    for zeros in (False, True):
        for dt in (L.F16, L.F32):
            q4_check(*q4_case(600, N, group, dt, vectors, zeros, L.BF16, seed=N), N, group, dt, dt_s=L.BF16)


# ------------------------------------------------------------------------------------------------
# The paged cache
# ------------------------------------------------------------------------------------------------

class Pages:
    """A cache with a page table whose pages are in no order, in one of several layouts."""

    def __init__(self, dt, seqs, width, page, heads, D, layout="dense", seed=0, spare=3):
        g = gen(seed)
        n = seqs * width + spare
        self.dt, self.page, self.heads, self.D, self.num_pages, self.width, self.seqs = dt, page, heads, D, n, width, seqs
        self.table = torch.randperm(n, device="cuda", generator=g)[: seqs * width].to(torch.int32).view(seqs, width).contiguous()
        if layout == "dense":
            self.k, self.v = (normal(g, dt, n, page, heads, D) for _ in range(2))
        elif layout == "heads first":  # [page][head][slot][dim]
            self.k, self.v = (normal(g, dt, n, heads, page, D).transpose(1, 2) for _ in range(2))
        elif layout == "together":  # keys and values of a page side by side, slots padded
            both = normal(g, dt, n, 2, page, heads * D + 8)
            self.k, self.v = (both[:, i, :, : heads * D].unflatten(-1, (heads, D)) for i in range(2))
        else:  # "odd": rows on no 16-byte boundary
            both = [normal(g, dt, n, page, heads, D + 1) for _ in range(2)]
            self.k, self.v = (t[..., 1:] for t in both)

    def cache(self):
        return L.KvCache(self.k, self.v, self.dt, self.num_pages, self.page, self.heads, self.D,
                         k_strides=self.k.stride()[:3], v_strides=self.v.stride()[:3])

    def rows(self, b, lo, hi):
        at = torch.arange(lo, hi, device="cuda")
        p = self.table[b].long()[at // self.page]
        return self.k[p, at % self.page], self.v[p, at % self.page]


LAYOUTS = ["dense", "heads first", "together", "odd"]


def attn_exact(P, q, lens, scale, window, dt):
    """(out, lse, slack of out, slack of lse) in 64 bits."""
    B, H, D = q.shape
    G = H // P.heads
    out, lse = torch.zeros(B, H, D, dtype=torch.float64, device="cuda"), torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    s_out, s_lse = torch.zeros_like(out), torch.zeros_like(out[..., 0])
    u16 = {L.F32: 0.0, L.F16: 2.0 ** -11, L.BF16: 2.0 ** -8}[dt]
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        k, v = (t.double() for t in P.rows(b, lo, n))
        qq = q[b].double().view(P.heads, G, D)
        score = torch.einsum("hgd,nhd->hgn", qq, k) * scale
        d = (2 * U * (D + 8) * abs(scale) * torch.einsum("hgd,nhd->hgn", qq.abs(), k.abs())).amax(-1)
        l = torch.logsumexp(score, -1)
        w = torch.exp(score - l[..., None])
        out[b] = torch.einsum("hgn,nhd->hgd", w, v).reshape(H, D)
        rel = 2 * d + 2.0 ** -20 + u16 + 2 * U * (160 + (n - lo) / 16)
        s_out[b] = (rel[..., None] * torch.einsum("hgn,nhd->hgd", w, v.abs())).reshape(H, D)
        lse[b] = l.reshape(H)
        s_lse[b] = (d + 2.0 ** -20 + 2 * U * (160 + (n - lo) / 16)).reshape(H)
    return out, lse, s_out, s_lse


def attn_check(P, lens, heads_q, dt, window=0, scale=0.0, seed=1, stream=None, plan=None, q_pad=0):
    B = len(lens)
    q = normal(gen(seed), dt, B, heads_q * P.D + q_pad)
    out = torch.full((B, heads_q * P.D + q_pad), math.nan, dtype=TORCH[dt], device="cuda")
    lse = torch.full((B, heads_q), math.nan, device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    plan = plan or L.PagedAttention(P.cache(), P.table, P.seqs, P.width, heads_q, scale=scale, window=window,
                                    q_token=heads_q * P.D + q_pad, out_token=heads_q * P.D + q_pad)
    plan.decode(q, out, n, B, lse=lse, stream=stream)
    torch.cuda.synchronize()
    q3 = q[:, : heads_q * P.D].unflatten(-1, (heads_q, P.D))
    want, want_lse, s_out, s_lse = attn_exact(P, q3, lens, scale or 1 / math.sqrt(P.D), window, dt)
    close(out[:, : heads_q * P.D].unflatten(-1, (heads_q, P.D)), want, s_out, dt)
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all()
    close(lse[~empty], want_lse[~empty], s_lse[~empty], L.F32)
    assert torch.isnan(out[:, heads_q * P.D:]).all()
    return out, lse


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("heads,G", [(1, 1), (3, 2), (2, 5), (2, 8), (1, 12), (2, 16), (1, 33)])
def test_attention_head_layouts(dt, heads, G):
    P = Pages(dt, 5, 20, 16, heads, 64, seed=G)
    attn_check(P, [300, 0, 1, 17, 255], heads * G, dt)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("D", [1, 8, 33, 40, 72, 80, 96, 100, 112, 128, 160, 192, 250, 256])
def test_attention_head_sizes(dt, D):
    P = Pages(dt, 3, 14, 16, 2, D, seed=D)
    attn_check(P, [200, 33, 7], 6, dt)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("page", [1, 7, 64])
def test_attention_layouts_and_pages(dt, layout, page):
    width = -(-230 // page)
    P = Pages(dt, 4, width, page, 2, 64, layout, seed=page)
    attn_check(P, [230, 65, 64, 63], 8, dt, q_pad=0 if layout == "dense" else 3)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("window", [1, 15, 64, 100, 5000])
def test_attention_window(dt, window):
    P = Pages(dt, 6, 40, 16, 2, 128, seed=window)
    attn_check(P, [640, 100, 101, 16, 1, 0], 8, dt, window=window)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("lens", [[5000], [4097, 1], [0, 9000, 3, 2048, 1, 0, 777], [40000], [0], [64] * 40])
def test_attention_lengths(dt, lens):
    page = 32
    P = Pages(dt, len(lens), max(1, -(-max(lens) // page)), page, 2, 64, seed=len(lens))
    first = attn_check(P, lens, 4, dt)
    again = attn_check(P, lens, 4, dt)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])  # the same bits every time


def test_attention_many_sequences():
    lens = [(37 * i) % 200 for i in range(700)]
    P = Pages(L.BF16, 700, 13, 16, 1, 64, seed=8)
    attn_check(P, lens, 4, L.BF16)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("D", [64, 160])
@pytest.mark.parametrize("seqs", [1, 5, 40, 150])
def test_attention_short_and_long_sequences_in_one_batch(dt, D, seqs):
    """Heads that one block does whole next to heads that are cut, from fewer to many more than there are blocks."""
    tile = 128 if D <= 128 and dt == L.BF16 else 64 if dt == L.BF16 or D <= 128 else 32
    some = [1, tile, 0, 3 * tile, 3 * tile + 1, tile + 1, 12 * tile + 5, 0, 0, 4 * tile, 2 * tile - 1]
    lens = [some[(i * i + 3) % len(some)] for i in range(seqs)]
    P = Pages(dt, seqs, -(-max(max(lens), 1) // 16), 16, 3, D, seed=seqs)
    for scale in (0.0, -0.25):
        first = attn_check(P, lens, 6, dt, scale=scale)
        again = attn_check(P, lens, 6, dt, scale=scale)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_attention_slots_past_the_end_may_hold_anything(dt):
    P = Pages(dt, 4, 10, 16, 2, 64, seed=3)
    lens, window = [150, 33, 0, 16], 40
    want = attn_check(P, lens, 8, dt, window=window)
    for b, n in enumerate(lens):
        at = torch.tensor([p for p in range(160) if p >= n or p < n - window], device="cuda")
        rows = P.table[b].long()[at // 16], at % 16
        P.k[rows], P.v[rows] = math.nan, -math.inf
    P.table[1, 3:] = -1
    P.table[2, :] = 1 << 30
    got = attn_check(P, lens, 8, dt, window=window)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("page", [16, 10])
def test_attention_does_not_look_up_pages_before_the_window(dt, page):
    """A sliding window's old pages may have been given back: their entries are never used."""
    P = Pages(dt, 3, 40, page, 2, 64, seed=13)
    lens, window = [390, 200, 77], 50
    want = attn_check(P, lens, 4, dt, window=window)
    for b, n in enumerate(lens):
        P.table[b, : (n - window) // page] = -1
        P.table[b, -(-n // page):] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    plan = L.PagedAttention(P.cache(), P.table, P.seqs, P.width, 4, window=window, status=status)
    got = attn_check(P, lens, 4, dt, window=window, plan=plan)
    assert status.item() == 0 and torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
def test_cache_without_pages_reports_every_key(dt):
    """A table that points into a cache of no pages: nothing is read, the rows are empty and the status says so."""
    table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = L.KvCache(None, None, dt, 0, 16, 1, 64)
    q, lens = normal(gen(1), dt, 2, 2, 64), torch.tensor([40, 0], dtype=torch.int32, device="cuda")
    out, lse = torch.ones_like(q), torch.zeros(2, 2, device="cuda")
    L.PagedAttention(cache, table, 2, 3, 2, status=status).decode(q, out, lens, 2, lse=lse)
    torch.cuda.synchronize()
    assert status.item() == L.KV_BAD_PAGE and (out == 0).all() and (lse == -math.inf).all()
    status.zero_()
    k = normal(gen(2), dt, 2, 1, 64)
    L.KvAppend(cache, table, 2, 3, status=status).append(k, k, lens, 2)
    torch.cuda.synchronize()
    assert status.item() == L.KV_BAD_PAGE


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_attention_infinities_and_nans_in_live_keys(dt):
    P = Pages(dt, 4, 6, 16, 1, 64, seed=4)
    q = torch.ones(4, 2, 64, dtype=TORCH[dt], device="cuda")
    lens = torch.tensor([90, 90, 90, 90], dtype=torch.int32, device="cuda")

    def slot(b, p):
        return int(P.table[b, p // 16]), p % 16

    P.k[slot(0, 40)] = -math.inf  # a key nobody attends to
    for p in range(90):
        P.k[slot(1, p)] = -math.inf  # no key has a score
    P.k[slot(2, 5)] = math.nan
    P.v[slot(3, 5)][0, 3] = math.nan  # one element of one value
    out, lse = torch.empty_like(q), torch.empty(4, 2, device="cuda")
    L.PagedAttention(P.cache(), P.table, 4, 6, 2).decode(q, out, lens, 4, lse=lse)
    k, v = (t[:, 0].double() for t in P.rows(0, 0, 90))
    s = (k @ q[0, 0].double()) / 8.0
    close(lse[0], torch.logsumexp(s, 0).expand(2), 1e-5 * torch.ones(2, device="cuda", dtype=torch.float64), L.F32)
    assert torch.isfinite(out[0]).all()
    assert torch.equal(out[1], torch.zeros_like(out[1])) and (lse[1] == -math.inf).all()
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all()
    assert torch.isnan(out[3][:, 3]).all() and torch.isfinite(out[3][:, :3]).all() and torch.isfinite(out[3][:, 4:]).all()


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
def test_attention_large_scores(dt):
    """Scores of thousands, of either sign, and a negative scale: the largest one decides, nothing overflows."""
    P = Pages(dt, 2, 20, 16, 2, 64, seed=5)
    P.k.mul_(64)
    attn_check(P, [300, 31], 4, dt, scale=0.25)
    attn_check(P, [300, 31], 4, dt, scale=-0.25)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
def test_attention_reports_bad_pages_and_leaves_them_out(dt):
    P = Pages(dt, 3, 8, 16, 1, 64, seed=6)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, lens = normal(gen(1), dt, 3, 2, 64), torch.tensor([128, 100, 1000], dtype=torch.int32, device="cuda")
    P.table[0, 2], P.table[0, 5] = -1, P.num_pages
    out = torch.empty_like(q)
    plan = L.PagedAttention(P.cache(), P.table, 3, 8, 2, status=status)
    plan.decode(q, out, lens, 2)
    torch.cuda.synchronize()
    assert status.item() == L.KV_BAD_PAGE
    at = torch.tensor([p for p in range(128) if p // 16 not in (2, 5)], device="cuda")
    rows = P.table[0].long()[at // 16], at % 16
    k, v = P.k[rows][:, 0].double(), P.v[rows][:, 0].double()
    want = torch.softmax(q[0].double() @ k.t() / 8.0, -1) @ v
    assert (out[0].double() - want).abs().max() < (1e-5 if dt == L.F32 else 2e-2)
    status.zero_()
    plan.decode(q[1:], out[1:], lens[1:], 1)  # row 0 of the table again, all its keys
    torch.cuda.synchronize()
    assert status.item() == L.KV_BAD_PAGE  # 100 keys reach page 5
    P.table[0, 2], P.table[0, 5] = 0, 1
    status.zero_()
    plan.decode(q, out, torch.tensor([128, -5, 1000], dtype=torch.int32, device="cuda"), 3)
    torch.cuda.synchronize()
    assert status.item() == L.KV_BAD_PAGE  # 1000 keys, a table of 128
    assert torch.equal(out[1], torch.zeros_like(out[1]))
    k, v = (t[:, 0].double() for t in P.rows(2, 0, 128))
    want = torch.softmax(q[2].double() @ k.t() / 8.0, -1) @ v
    assert (out[2].double() - want).abs().max() < (1e-5 if dt == L.F32 else 2e-2)


def test_cache_offsets_pass_32_bits():
    """Pages four billion elements apart: the append writes there and the attention reads there."""
    page, heads, D, n = 16, 1, 64, 2
    stride = (1 << 32) + 1024
    buf = torch.empty(stride + 2 * page * heads * D, dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    strides = (stride, heads * D, D)
    cache = L.KvCache(buf, buf[page * heads * D:], L.BF16, n, page, heads, D, k_strides=strides, v_strides=strides)
    g = gen(9)
    k, v, q = normal(g, L.BF16, 20, heads, D), normal(g, L.BF16, 20, heads, D), normal(g, L.BF16, 1, 2, D)
    pos, seq = torch.arange(20, dtype=torch.int32, device="cuda"), torch.zeros(20, dtype=torch.int32, device="cuda")
    L.KvAppend(cache, table, 1, 2).append(k, v, pos, 20, seq=seq)
    out = torch.empty_like(q)
    L.PagedAttention(cache, table, 1, 2, 2).decode(q, out, torch.tensor([20], dtype=torch.int32, device="cuda"), 1)
    torch.cuda.synchronize()
    assert torch.equal(buf[stride: stride + page * D].view(page, D), k[:16, 0])
    assert torch.equal(buf[page * D: page * D + 4 * D].view(4, D), v[16:, 0])
    want = torch.softmax(q[0].double() @ k[:, 0].double().t() / 8.0, -1) @ v[:, 0].double()
    assert (out[0].double() - want).abs().max() < 2e-2


# ------------------------------------------------------------------------------------------------
# Append
# ------------------------------------------------------------------------------------------------

def turned(x, cos, sin, rot, interleaved):
    """(rotated, slack) of [tokens][heads][D] in 64 bits."""
    y, slack = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    if rot:
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        c, s = cos.double()[:, None, :], sin.double()[:, None, :]
        u, w = x.double()[..., a], x.double()[..., b]
        y[..., a], y[..., b] = u * c - w * s, w * c + u * s
        slack[..., a] = slack[..., b] = 4 * U * (u.abs() + w.abs())
    return y, slack


def append_check(P, seq, pos, heads_q, rot, interleaved, dt, pad=0, in_place=False, shift=0, stream=None):
    T, D, g = len(pos), P.D, gen(len(pos) + rot)
    cos, sin = L.rotation_tables(max(pos) + 1, rot, device="cuda") if rot else (None, None)
    if rot and shift:
        cos, sin = offset_view(cos, 1), offset_view(sin, 1)

    def token_rows(h):
        t = normal(g, dt, T, h * D + pad)
        t = offset_view(t, shift) if shift else t
        return t, t[:, : h * D].unflatten(-1, (h, D))

    (k_raw, k), (v_raw, v), (q_raw, q) = token_rows(P.heads), token_rows(P.heads), token_rows(max(heads_q, 1))
    q0 = q.clone()
    qo_raw = q_raw if in_place else torch.full_like(q_raw, -7.0)
    qo = qo_raw[:, : max(heads_q, 1) * D].unflatten(-1, (max(heads_q, 1), D))
    k_was, v_was = P.k.clone(), P.v.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    op = L.KvAppend(P.cache(), P.table, P.seqs, P.width, heads_q=heads_q, cos=cos, sin=sin, max_pos=max(pos) + 1, rot_dim=rot,
                    interleaved=interleaved, k_token=P.heads * D + pad, v_token=P.heads * D + pad,
                    q_token=heads_q * D + pad if heads_q else 0, q_out_token=heads_q * D + pad if heads_q else 0, status=status)
    pos_d = torch.tensor(pos, dtype=torch.int32, device="cuda")
    seq_d = None if seq is None else torch.tensor(seq, dtype=torch.int32, device="cuda")
    op.append(k_raw, v_raw, pos_d, T, seq=seq_d, q=q_raw if heads_q else None, q_out=qo_raw if heads_q else None, stream=stream)
    torch.cuda.synchronize()
    assert status.item() == 0
    live = torch.nonzero(pos_d >= 0)[:, 0]
    at, of = pos_d[live].long(), live if seq is None else seq_d[live].long()
    where = P.table.long()[of, at // P.page], at % P.page
    c, s = (cos[at], sin[at]) if rot else (None, None)
    want, slack = turned(k[live], c, s, rot, interleaved)
    close(P.k[where], want, slack, dt)
    assert torch.equal(P.v[where], v[live])
    assert torch.equal(P.k[where][..., rot:], k[live][..., rot:])
    k_was[where], v_was[where] = P.k[where], P.v[where]
    assert torch.equal(P.k, k_was) and torch.equal(P.v, v_was)  # every other slot as it was
    if heads_q:
        want, slack = turned(q0[live], c, s, rot, interleaved)
        close(qo[live], want, slack, dt)
        dead = torch.nonzero(pos_d < 0)[:, 0]
        assert torch.equal(qo[dead], q0[dead] if in_place else torch.full_like(q0[dead], -7.0))
        if pad and not in_place:
            assert (qo_raw[:, heads_q * D:] == -7.0).all()


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (80, 32), (64, 0), (66, 34), (33, 2), (2, 2), (256, 256), (48, 48)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_rotations(dt, D, rot, interleaved):
    append_check(Pages(dt, 3, 5, 16, 2, D, seed=D), [0] * 40 + [2] * 9, list(range(20, 60)) + list(range(9)), 6, rot, interleaved, dt)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("pad,shift,in_place", [(0, 0, True), (8, 0, False), (3, 0, True), (0, 1, False)])
def test_append_layouts(dt, layout, pad, shift, in_place):
    P = Pages(dt, 4, 6, 7, 3, 64, layout, seed=pad)
    append_check(P, [3] * 10 + [1] * 5, list(range(30, 40)) + [0, 1, -1, 2, 41], 3, 64, False, dt, pad, in_place, shift)


@pytest.mark.parametrize("tokens", [1, 2, 31, 700])
def test_append_one_token_per_sequence(tokens):
    P = Pages(L.BF16, tokens, 3, 16, 2, 64, seed=tokens)
    pos = [(29 * i) % 48 for i in range(tokens)]
    if tokens > 2:
        pos[1] = -3
    append_check(P, None, pos, 4, 64, False, L.BF16)


def test_append_keys_and_values_only_and_page_size_one():
    append_check(Pages(L.F16, 2, 50, 1, 2, 64), [1] * 50, list(range(50)), 0, 64, False, L.F16)


def test_append_reports_and_leaves_out_bad_tokens():
    P = Pages(L.BF16, 2, 4, 16, 1, 64, seed=7)
    k_was = P.k.clone()
    k, v = normal(gen(1), L.BF16, 5, 1, 64), normal(gen(2), L.BF16, 5, 1, 64)
    cos, sin = L.rotation_tables(50, 64, device="cuda")
    q = normal(gen(3), L.BF16, 5, 2, 64)
    for pos, seq, bit, good in [([64, 0, 0, -1, -1], [0, 2, -1, 9, 0], L.KV_BAD_PAGE, []),
                                ([50, 3, 63, -9, -1], [0, 1, 1, 0, 0], L.KV_BAD_POSITION, [1])]:
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        qo = torch.zeros_like(q)
        L.KvAppend(P.cache(), P.table, 2, 4, heads_q=2, cos=cos, sin=sin, max_pos=50 if good else 1000, rot_dim=64 if good else 0,
                   status=status).append(k, v, torch.tensor(pos, dtype=torch.int32, device="cuda"), 5, q=q, q_out=qo,
                                         seq=torch.tensor(seq, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert status.item() == bit
        same = torch.ones(P.k.shape[:2], dtype=torch.bool, device="cuda")
        for t in good:
            same[int(P.table[seq[t], pos[t] // 16]), pos[t] % 16] = False
        assert torch.equal(P.k[same], k_was[same])
        for t in range(5):
            assert (qo[t] != 0).any() == (t in good)


# ------------------------------------------------------------------------------------------------
# Streams and graphs
# ------------------------------------------------------------------------------------------------

def test_operators_follow_their_stream():
    """Inputs written and outputs read on another stream, with no synchronisation in between."""
    s = torch.cuda.Stream()
    w, sc, z, x = q4_case(3000, 8192, 128, L.F16, 1, seed=1)
    P = Pages(L.F16, 2, 200, 16, 2, 64, seed=2)
    torch.cuda.synchronize()
    m, y = L.Q4Matrix(w, sc, 3000, 8192, 128), torch.zeros(1, 3000, dtype=torch.float16, device="cuda")
    plan = L.PagedAttention(P.cache(), P.table, 2, 200, 4)
    q, out, lens = normal(gen(3), L.F16, 2, 4, 64), torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda"), torch.tensor([3200, 50], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            big = big @ big * 1e-3
        x.mul_(2.0)
        m.gemv(x, y, stream=s)
        y2 = y * 1.0
        q.mul_(0.5)
        plan.decode(q, out, lens, 2, stream=s)
        out2 = out * 1.0
    s.synchronize()
    want, total = q4_exact(w, sc, z, x, 8192, 128)
    close(y2, want, 2 * U * (160 + 8192 / 32) * total, L.F16)
    want, _, slack, _ = attn_exact(P, q, [3200, 50], 0.125, 0, L.F16)
    close(out2, want, slack, L.F16)


def test_operators_in_a_graph():
    """A captured step (append, attention, product) replays with new lengths and inputs in its buffers."""
    dt, B, H, HK, D = L.BF16, 3, 4, 2, 64
    P = Pages(dt, B, 20, 16, HK, D, seed=11)
    cos, sin = L.rotation_tables(320, D, device="cuda")
    qkv = normal(gen(1), dt, B, (H + 2 * HK) * D)
    row = qkv.shape[1]
    ap = L.KvAppend(P.cache(), P.table, B, 20, heads_q=H, cos=cos, sin=sin, max_pos=320, rot_dim=D, k_token=row, v_token=row, q_token=row, q_out_token=row)
    plan = L.PagedAttention(P.cache(), P.table, B, 20, H, q_token=row)
    w, sc, z, _ = q4_case(200, H * D, 64, dt, seed=2)
    m = L.Q4Matrix(w, sc, 200, H * D, 64, dtype_x=dt)
    pos, lens = torch.tensor([5, 200, 0], dtype=torch.int32, device="cuda"), torch.tensor([6, 201, 1], dtype=torch.int32, device="cuda")
    out, y = torch.zeros(B, H, D, dtype=TORCH[dt], device="cuda"), torch.zeros(B, 200, dtype=TORCH[dt], device="cuda")

    def step(stream):
        q, k, v = qkv, qkv[:, H * D:], qkv[:, (H + HK) * D:]
        ap.append(k, v, pos, B, q=q, q_out=q, stream=stream)
        plan.decode(q, out, lens, B, stream=stream)
        m.gemv(out, y, vectors=B, stream=stream)

    first = qkv.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(s)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream())
    for n in range(4):
        new = first * (n + 1)
        pos.add_(1)
        lens.add_(1)
        qkv.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), y.clone(), qkv.clone()
        qkv.copy_(new)
        step(None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (out, y, qkv)))
    assert np.isfinite(y.float().cpu().numpy()).all()
    del graph
