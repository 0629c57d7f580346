"""The decoding operators where 32-bit arithmetic has to be kept: sums whose largest terms cancel, weigh nothing or
lie far above the rest.

The tolerances come from rounding alone (u = 2^-24), with the bounds that test_decode_ops_gpu.py derives:

* q4: 2u (160 + n / 32) S, S the sum of the terms' absolute values; what has the weight zero adds nothing to S.
* attention: scores here are single products, exact but for the scale (two roundings, 2u |score|); a weight is off
  by 2^-20 for exp and by what its two 16-bit parts leave: 2^-16 of it for bf16; for fp16 2^-22 of it or 2^-39 of the
  largest weight, whichever is more.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import l2domain_b200 as L  # noqa: E402
from test_decode_ops_gpu import TORCH, U, Pages, attn_check, close, gen, gpu, normal, q4_exact  # noqa: E402,F401


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------

def steered(P, n, heads_q, dt, scores, values, q0):
    """Attention over n keys of each head whose only non-zero element is the first: key p of every head has the score
    q0[h] * scores[p] (scale 1).  (out, lse, want, want lse, slack, slack of lse) for one sequence."""
    D = P.D
    q = torch.zeros(1, heads_q, D, dtype=TORCH[dt], device="cuda")
    q[0, :, 0] = q0.to(TORCH[dt])
    at = torch.arange(n, device="cuda")
    rows = P.table[0].long()[at // P.page], at % P.page
    P.k[rows] = 0
    keys = torch.zeros(n, P.heads, D, dtype=TORCH[dt], device="cuda")
    keys[:, :, 0] = scores.to(TORCH[dt])[:, None]
    P.k[rows], P.v[rows] = keys, values.to(TORCH[dt])
    out = torch.full_like(q, math.nan)
    lse = torch.full((1, heads_q), math.nan, device="cuda")
    L.PagedAttention(P.cache(), P.table, P.seqs, P.width, heads_q, scale=1.0).decode(
        q, out, torch.tensor([n], dtype=torch.int32, device="cuda"), 1, lse=lse)
    torch.cuda.synchronize()
    k, v = (t.double().repeat_interleave(heads_q // P.heads, 1) for t in P.rows(0, 0, n))
    s = torch.einsum("hd,nhd->hn", q[0].double(), k)
    l = torch.logsumexp(s, -1)
    w = torch.exp(s - l[:, None])
    off = 2 * U * s.abs().amax(-1, keepdim=True) * 2 + 2.0 ** -20 + 2 * U * (160 + n / 16)
    part = {L.F32: 0 * w, L.BF16: w * 2.0 ** -16, L.F16: torch.maximum(w * 2.0 ** -22, w.amax(-1, keepdim=True) * 2.0 ** -39)}[dt]
    slack = torch.einsum("hn,nhd->hd", w * off + part, v.abs())
    return out[0], lse[0], torch.einsum("hn,nhd->hd", w, v), l, slack, off[:, 0]


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("G,D", [(2, 64), (16, 64), (1, 128), (5, 256), (12, 128)])
@pytest.mark.parametrize("power", [14, 27, 31, 36])
def test_attention_scores_far_apart(dt, G, D, power):
    """Scores of up to 2^power, each key's far below the next one's: the largest takes all, whatever the rounding of the
    others is worth."""
    power = min(power, 30) if dt == L.F16 else power
    P = Pages(dt, 1, 20, 16, 2, D, seed=power)
    n = 300
    low = min(power - power // 2, 15)
    scores = (torch.randperm(n, device="cuda", generator=gen(power)) + 1).float() * 2.0 ** (low - 9)
    scores = scores.to(TORCH[dt]).float()  # rounded: several may be the largest
    q0 = torch.full((2 * G,), 2.0 ** (power - low), device="cuda")
    g = gen(G)
    values = normal(g, dt, n, 2, D)
    top = torch.nonzero(scores == scores.max())[:, 0]
    values[top] = values[top[:1]].clone()
    out, lse, want, want_lse, _, _ = steered(P, n, 2 * G, dt, scores, values, q0)
    close(out, want, 2.0 ** -15 * want.abs(), dt)
    close(lse, want_lse, 2.0 ** -20 * want_lse.abs(), L.F32)


@pytest.mark.parametrize("G,D", [(1, 64), (8, 128), (12, 64), (16, 128), (16, 256), (33, 80)])
@pytest.mark.parametrize("nats", [8, 12, 18])
def test_attention_keeps_small_weights(G, D, nats):
    """A key far above the others whose values are zero: what comes out is all of the others'."""
    for dt in (L.F16, L.BF16):
        P = Pages(dt, 1, 30, 16, 1, D, seed=nats)
        n = 450
        g = gen(nats)
        scores = -(torch.rand(n, device="cuda", generator=g) + nats)
        scores[7] = 0.0
        values = normal(g, L.F32, n, 1, D).abs() * 500 + 100
        values[7] = 0.0
        q0 = torch.linspace(0.75, 1.0, G, device="cuda")
        out, lse, want, want_lse, slack, off = steered(P, n, G, dt, scores, values, q0)
        close(out, want, slack, dt)
        close(lse, want_lse, off, L.F32)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("G,D", [(1, 128), (8, 64), (7, 256), (9, 128), (12, 64), (16, 80), (16, 96), (16, 128), (16, 192), (16, 256), (33, 128)])
def test_attention_values_that_cancel(dt, G, D):
    """Two keys of nearly the same score and opposite values, among others that weigh little: the difference of their
    weights comes out, which weights of 8 or 11 bits would not have."""
    P = Pages(dt, 1, 20, 16, 1, D, seed=G)
    n = 300
    scores = torch.full((n,), -40.0, device="cuda")
    scores[4], scores[6] = 0.0, -0.015625  # of one tile: weights are relative to the largest in it
    g = gen(D)
    values = normal(g, L.F32, n, 1, D)
    values[6] = -values[4]
    q0 = (torch.arange(G, device="cuda") + 1) / 64.0 + 0.5
    out, lse, want, want_lse, slack, off = steered(P, n, G, dt, scores, values, q0)
    close(out, want, slack, dt)
    close(lse, want_lse, off, L.F32)


@pytest.mark.parametrize("dt", [L.F16, L.BF16])
@pytest.mark.parametrize("D", [80, 96, 128, 192, 250, 256])
@pytest.mark.parametrize("G", [9, 16, 40])
def test_attention_large_groups_on_wide_heads(dt, D, G):
    P = Pages(dt, 3, 20, 16, 2, D, seed=G)
    attn_check(P, [300, 0, 129], 2 * G, dt)


@pytest.mark.parametrize("D", [136, 160, 200, 256])
@pytest.mark.parametrize("G", [1, 5, 8, 17])
def test_attention_fp32_groups_on_wide_heads(D, G):
    P = Pages(L.F32, 3, 20, 16, 2, D, seed=G)
    attn_check(P, [300, 0, 129], 2 * G, L.F32)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("G,D", [(1, 64), (8, 128), (16, 64), (4, 256)])
def test_attention_values_near_the_end_of_the_range(dt, G, D):
    """Their mean is in the range, and their sum is not."""
    P = Pages(dt, 1, 130, 16, 1, D, seed=G)
    n = 2000
    largest = torch.finfo(TORCH[dt]).max
    scores = torch.rand(n, device="cuda", generator=gen(D)) * 0.25
    values = (0.5 + 0.25 * torch.rand(n, 1, D, device="cuda", generator=gen(G))) * largest
    values[:, :, 1::2] *= -1
    out, lse, want, want_lse, slack, off = steered(P, n, G, dt, scores, values, torch.ones(G, device="cuda"))
    close(out, want, slack, dt)
    close(lse, want_lse, off, L.F32)


def test_attention_large_scores_fp16():
    P = Pages(L.F16, 2, 20, 16, 2, 64, seed=5)
    P.k.mul_(64)
    for scale in (0.25, -0.25):
        attn_check(P, [300, 31], 4, L.F16, scale=scale)
        attn_check(P, [300, 31], 24, L.F16, scale=scale)


# ------------------------------------------------------------------------------------------------
# 4-bit products
# ------------------------------------------------------------------------------------------------

def product(w, s, z, x, N, group, dt, dt_y):
    M, vectors = w.shape[0], x.shape[0]
    y = torch.full((vectors, M), math.nan, dtype=TORCH[dt_y], device="cuda")
    L.Q4Matrix(w, s, M, N, group, zeros=z, dtype_x=dt, dtype_y=dt_y, ldw=w.stride(0), lds=s.stride(0)).gemv(x, y, vectors=vectors, stride_x=x.stride(0))
    torch.cuda.synchronize()
    return y


def weights(M, N, group, zeros, seed, pad=0):
    g = gen(seed)
    groups = -(-N // group)
    w = torch.randint(0, 256, (M, (N + 1) // 2 + pad), dtype=torch.uint8, device="cuda", generator=g)
    s = torch.empty(M, groups, device="cuda").uniform_(0.01, 0.02, generator=g).half()
    z = torch.randint(0, 16, (M, groups), dtype=torch.uint8, device="cuda", generator=g) if zeros else None
    return w, s, z


def set_weight(w, column, value):
    """q of a column of every row."""
    byte, shift = w[:, column // 2], 4 * (column % 2)
    w[:, column // 2] = (byte & (0xF0 if shift == 0 else 0x0F)) | (value.to(torch.uint8) << shift)


def zero_point(z, column, group, M):
    return z[:, column // group] & 15 if z is not None else torch.full((M,), 8, dtype=torch.uint8, device="cuda")


def tolerance(N, total):
    return 2 * U * (160 + N / 32) * total


LARGE = [(L.F32, L.F32, 1e4), (L.F32, L.F32, 1e6), (L.F32, L.F32, 2.0 ** 32), (L.F32, L.F32, 1e10), (L.F32, L.F32, 1e30),
         (L.BF16, L.F32, 1e6), (L.BF16, L.F32, 1e12), (L.BF16, L.BF16, 1e8), (L.BF16, L.BF16, 3e35), (L.F16, L.F32, 6e4),
         (L.F16, L.F16, 6e4), (L.F32, L.BF16, 1e9)]


def large_activation(dt, dt_y, large, group, vectors):
    """What the largest activation is multiplied with is zero: the others have all their bits."""
    M, N = 70, 1152
    w, s, z = weights(M, N, group, group == 64, seed=group)
    x = normal(gen(3), L.F32, vectors, N)
    if dt == L.F16:
        x *= 0.01
    for b in range(vectors):
        for column in (5 + 17 * b, 640 + b):
            set_weight(w, column, zero_point(z, column, group, M))
            x[b, column] = -large if b % 2 else large
    x = x.to(TORCH[dt])
    want, total = q4_exact(w, s, z, x, N, group)
    close(product(w, s, z, x, N, group, dt, dt_y), want, tolerance(N, total), dt_y)


def every_size(dt, group, vectors):
    """Powers of two from 2^-40 to 2^40 in one vector, the largest on weights of zero; and all of them scaled by 2^60."""
    M, N = 33, 1024
    w, s, z = weights(M, N, group, True, seed=vectors)
    g = gen(5)
    size = torch.randint(-40, 41, (vectors, N), device="cuda", generator=g).float()
    x = normal(g, L.F32, vectors, N) * torch.exp2(size)
    for column in torch.unique(torch.nonzero(size > 0)[:, 1]).tolist():
        set_weight(w, column, zero_point(z, column, group, M))
    for scale in (1.0, 2.0 ** 60, 2.0 ** -60):
        xx = (x * scale).to(TORCH[dt])
        want, total = q4_exact(w, s, z, xx, N, group)
        close(product(w, s, z, xx, N, group, dt, L.F32), want, tolerance(N, total), L.F32)


@pytest.mark.parametrize("dt,dt_y,large", LARGE)
@pytest.mark.parametrize("group", [32, 64, 128, 384])
@pytest.mark.parametrize("vectors", [3, 9])
def test_q4_large_activation_on_a_zero_weight_several_vectors(dt, dt_y, large, group, vectors):
    large_activation(dt, dt_y, large, group, vectors)


@pytest.mark.parametrize("dt,dt_y,large", LARGE)
@pytest.mark.parametrize("group", [32, 64, 128, 384])
@pytest.mark.parametrize("vectors", [1, 2])
def test_q4_large_activation_on_a_zero_weight(dt, dt_y, large, group, vectors):
    large_activation(dt, dt_y, large, group, vectors)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("group", [32, 64, 128, 512])
def test_q4_activations_of_every_size_several_vectors(dt, group):
    every_size(dt, group, 4)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("group", [32, 64, 128, 512])
@pytest.mark.parametrize("vectors", [1, 2])
def test_q4_activations_of_every_size(dt, group, vectors):
    every_size(dt, group, vectors)


@pytest.mark.parametrize("dt,dt_y", [(L.F32, L.F32), (L.F16, L.F16), (L.BF16, L.BF16), (L.BF16, L.F32)])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("vectors", [1, 2, 5])
def test_q4_rows_of_few_weights(dt, dt_y, group, vectors):
    """Rows with one weight that is not zero, and one with none: the other columns leave nothing behind."""
    M, N = 40, 768
    w, s, z = weights(M, N, group, group == 256, seed=7)
    for column in range(N):
        set_weight(w, column, zero_point(z, column, group, M))
    for row in range(1, M):
        column = 19 * row
        q = int(w[row, column // 2]) ^ (7 << (4 * (column % 2)))
        w[row, column // 2] = q
    x = normal(gen(8), L.F32, vectors, N)
    x[:, 19 * 3] = 0.0078125
    x = x.to(TORCH[dt])
    want, total = q4_exact(w, s, z, x, N, group)
    y = product(w, s, z, x, N, group, dt, dt_y)
    assert (y[:, 0] == 0).all()
    close(y, want, tolerance(N, total), dt_y)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("vectors", [1, 2, 5])
def test_q4_sums_that_pass_the_range_before_their_scale(dt, group, vectors):
    """Activations of 2^122: sums of (q - z) x pass the range of fp32, the scaled ones do not."""
    M, N = 20, 512
    w, s, z = weights(M, N, group, False, seed=9)
    w |= 0x88  # all weights positive
    s *= 2.0 ** -6
    x = ((normal(gen(2), L.F32, vectors, N).abs() + 1) * 2.0 ** 122).to(TORCH[dt])
    want, total = q4_exact(w, s, z, x, N, group)
    assert want.max() < 2.0 ** 127
    close(product(w, s, z, x, N, group, dt, dt), want, tolerance(N, total), dt)


def infinities_and_nans(dt, group, vectors):
    """They reach their own vector, beside activations of wide range, which keep their bits in the others."""
    M, N = 50, 640
    w, s, z = weights(M, N, group, True, seed=11)
    set_weight(w, 300, zero_point(z, 300, group, M))
    set_weight(w, 200, (zero_point(z, 200, group, M) + 1) % 16)  # z + 1, or -15 where z is 15
    x = normal(gen(4), L.F32, vectors, N).to(TORCH[dt])
    x[:, 300] = 60000.0
    clean = product(w, s, z, x, N, group, dt, L.F32)
    want, total = q4_exact(w, s, z, x, N, group)
    close(clean, want, tolerance(N, total), L.F32)
    last = vectors - 1
    for odd in (math.inf, -math.inf, math.nan):
        x[last, 200] = odd
        y = product(w, s, z, x, N, group, dt, L.F32)
        assert torch.equal(y[:last], clean[:last])
        up = zero_point(z, 200, group, M) != 15
        assert torch.isnan(y[last]).all() if math.isnan(odd) else torch.equal(y[last], torch.where(up, odd, -odd))


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("vectors", [3, 10])
def test_q4_infinities_and_nans_several_vectors(dt, group, vectors):
    infinities_and_nans(dt, group, vectors)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("vectors", [1, 2])
def test_q4_infinities_and_nans(dt, group, vectors):
    infinities_and_nans(dt, group, vectors)


@pytest.mark.parametrize("dt,dt_y", [(L.F32, L.F32), (L.F16, L.F16), (L.BF16, L.BF16), (L.F16, L.F32)])
@pytest.mark.parametrize("group", [32, 64, 128, 384])
def test_q4_vector_alone_and_in_company(dt, dt_y, group):
    """A vector by itself and the same one among eight: both within the rounding of the same sums."""
    M, N = 90, 1152
    w, s, z = weights(M, N, group, True, seed=13)
    x = normal(gen(6), dt, 8, N)
    want, total = q4_exact(w, s, z, x, N, group)
    close(product(w, s, z, x, N, group, dt, dt_y), want, tolerance(N, total), dt_y)
    for b in range(8):
        close(product(w, s, z, x[b:b + 1], N, group, dt, dt_y), want[b:b + 1], tolerance(N, total[b:b + 1]), dt_y)
