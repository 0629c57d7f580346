"""The paged cache in 4 bits on the GPU: what an append stores, bit for bit, and attention over it against its definition in
64 bits.

Tolerances of the attention, per element, from rounding alone (u = 2^-24; a matrix instruction may truncate where it adds,
which costs twice a rounding): products of queries and 4-bit differences are exact, so a score is off by
d = 2u (D + 16) |scale| sum|q k|, a weight by a factor of at most 1 + 2 d and some 2^-20 for exp; a weight times a
scale meets the values as two bf16 numbers, which leaves 2^-16 of it, or as three (fp32), which leaves 2^-24; sums add
2u (160 + n / 16).  All of it is relative to sum w |v|.  On top, where the keys that decide have a 0 for a value and all
others next to no weight: a weight below 2^-126 is 0, and a weight times a scale times 2^-24 ends at bf16's last place, 2^-133,
so that each key may be off by 2^-126 |v| + 15 * 2^-109, for which 2^-104 (1 + |v|) stands (`least`).  Where scores are capped or biased, d grows by 8u (cap + the
largest bias and score), tanh being off by two units in the last place at most.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import l2domain_b200 as L  # noqa: E402
from test_decode_ops_gpu import TORCH, U, close, gen, gpu, normal, offset_view, turned  # noqa: E402,F401

FIFTEENTH = torch.tensor(1.0 / 15.0, dtype=torch.float32).double().item()


def once(x):
    """Of one operation on fp32 numbers, done in 64 bits: as fp32 rounds it."""
    return x.float().double()


def quantised(x, group):
    """(n, z, s) of [..][D] in 64 bits: the numbers, and zero points and scales of the groups."""
    ns, zs, ss = [], [], []
    for lo in range(0, x.shape[-1], group):
        g = x[..., lo: lo + group].double()
        least, most = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
        s = once(once(most * FIFTEENTH) - once(least * FIFTEENTH))
        bits = s.float().view(torch.int32)
        s = ((bits + 15) // 16 * 16).view(torch.float32).double()
        by = torch.where(s == 0, 1.0, s)
        z = torch.round(once(-least / by)).clamp(max=15.0)
        ns.append((torch.round(once(g / by[..., None])) + z[..., None]).clamp(0, 15))
        zs.append(z)
        ss.append(s)
    return torch.cat(ns, -1), torch.stack(zs, -1), torch.stack(ss, -1)


def stand_for(n, z, s, group):
    D = n.shape[-1]
    return s.repeat_interleave(group, -1)[..., :D] * (n - z.repeat_interleave(group, -1)[..., :D])


class Pages4:
    """A cache in 4 bits with a page table in no order; k and v [page][slot][head][D] are its values in 64 bits."""

    def __init__(self, dt, seqs, width, page, heads, D, group, seed=0, spare=2, together=False, scale=1.0):
        g = gen(seed)
        n = seqs * width + spare
        self.dt, self.page, self.heads, self.D, self.group, self.num_pages, self.width, self.seqs = dt, page, heads, D, group, n, width, seqs
        self.table = torch.randperm(n, device="cuda", generator=g)[: seqs * width].to(torch.int32).view(seqs, width).contiguous()
        self.bytes = L.kv4_page_bytes(page, heads, D, group)
        if together:  # keys and values of a page side by side, pages padded
            both = torch.randint(0, 256, (n, 2 * self.bytes + 16), dtype=torch.uint8, device="cuda", generator=g)
            self.raw = [both[:, : self.bytes], both[:, self.bytes: 2 * self.bytes]]
        else:
            self.raw = [torch.randint(0, 256, (n, self.bytes), dtype=torch.uint8, device="cuda", generator=g) for _ in range(2)]
        self.k, self.v = (torch.empty(n, page, heads, D, device="cuda").normal_(generator=g) * scale for _ in range(2))
        self.k[..., : D // 3] += scale  # groups of one sign more than the other
        self.parts = [self.fill(i, x) for i, x in enumerate((self.k, self.v))]
        self.k, self.v = (stand_for(*p, group) for p in self.parts)

    def views(self, raw):
        """Nibble bytes [page][block][head][32s][slot][16] and words [page][block][head][group][slot]."""
        chunks, groups = -(-self.D // 32), -(-self.D // self.group)
        t = raw.unflatten(1, (self.page // 16, self.heads, 256 * chunks + 64 * groups))
        return t[..., : 256 * chunks].unflatten(-1, (chunks, 16, 16)), t[..., 256 * chunks:].view(torch.int32).unflatten(-1, (groups, 16))

    def fill(self, which, x):
        n, z, s = quantised(x, self.group)
        number, word = self.packed(n, z, s)
        nibbles, words = self.views(self.raw[which])
        nibbles.copy_(number.unflatten(1, (-1, 16)).permute(0, 1, 3, 4, 2, 5))
        words.copy_(word.unflatten(1, (-1, 16)).permute(0, 1, 3, 4, 2))
        return n, z, s

    @staticmethod
    def packed(n, z, s):
        n = torch.nn.functional.pad(n, (0, -n.shape[-1] % 32)).to(torch.uint8)
        return (n[..., 0::2] + 16 * n[..., 1::2]).unflatten(-1, (-1, 16)), s.float().view(torch.int32) + z.int()

    def cache(self):
        return L.KvCache4(self.raw[0], self.raw[1], self.dt, self.num_pages, self.page, self.heads, self.D, self.group,
                          k_page=self.raw[0].stride(0), v_page=self.raw[1].stride(0))

    def rows(self, b, lo, hi):
        at = torch.arange(lo, hi, device="cuda")
        p = self.table[b].long()[at // self.page]
        return self.k[p, at % self.page], self.v[p, at % self.page]


def attention(P, q, lens, scale, window=0, cap=0.0, slopes=None, starts=None, parts=None, least=2.0 ** -104):
    """(out, lse, slack of out, slack of lse) in 64 bits; parts: what a weight loses on the way to the values, least: what it
    loses whatever its size."""
    B, H, D = q.shape
    G = H // P.heads
    out, lse = torch.zeros(B, H, D, dtype=torch.float64, device="cuda"), torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    s_out, s_lse = torch.zeros_like(out), torch.zeros_like(out[..., 0])
    for b, n in enumerate(lens):
        lo = max(0, n - window if window else 0, starts[b] if starts else 0)
        if n <= lo:
            continue
        k, v = (t.double() for t in P.rows(b, lo, n))
        qq = q[b].double().view(P.heads, G, D)
        score = torch.einsum("hgd,nhd->hgn", qq, k) * scale
        d = (2 * U * (D + 16) * abs(scale) * torch.einsum("hgd,nhd->hgn", qq.abs(), k.abs())).amax(-1)
        if cap:
            score = cap * torch.tanh(score / cap)
        bias = torch.zeros_like(score)
        if slopes is not None:
            bias = slopes.double().view(P.heads, G, 1) * torch.arange(lo - n + 1, 1, device="cuda").double()
            score = score + bias
        if cap or slopes is not None:
            d = d + 8 * U * (cap + (bias.abs() + score.abs()).amax(-1))
        l = torch.logsumexp(score, -1)
        w = torch.exp(score - l[..., None])
        out[b] = torch.einsum("hgn,nhd->hgd", w, v).reshape(H, D)
        rel = 2 * d + 2.0 ** -20 + parts + 2 * U * (160 + (n - lo) / 16)
        s_out[b] = (rel[..., None] * torch.einsum("hgn,nhd->hgd", w, v.abs())).reshape(H, D) + least * (n - lo) * (1 + v.abs().max())
        lse[b] = l.reshape(H)
        s_lse[b] = (d + 2.0 ** -20 + 2 * U * (160 + (n - lo) / 16)).reshape(H)
    return out, lse, s_out, s_lse


def check(P, lens, heads_q, dt, window=0, scale=0.0, cap=0.0, slopes=None, starts=None, seed=1, stream=None, plan=None, parts=None, least=2.0 ** -104, q=None):
    B = len(lens)
    q = normal(gen(seed), dt, B, heads_q, P.D) if q is None else q
    out = torch.full((B + 1, heads_q, P.D), math.nan, dtype=TORCH[dt], device="cuda")
    lse = torch.full((B + 1, heads_q), math.nan, device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    at = torch.tensor(starts, dtype=torch.int32, device="cuda") if starts else None
    plan = plan or L.PagedAttention(P.cache(), P.table, P.seqs, P.width, heads_q, scale=scale, window=window, cap=cap, slopes=slopes)
    plan.decode(q, out, n, B, lse=lse, stream=stream, starts=at)
    torch.cuda.synchronize()
    if parts is None:
        parts = 2.0 ** -24 if dt == L.F32 else 2.0 ** -16
    want, want_lse, s_out, s_lse = attention(P, q, lens, scale or 1 / math.sqrt(P.D), window, cap, slopes, starts, parts, least)
    close(out[:B], want, s_out, dt)
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse[:B]), empty) and (lse[:B][empty] < 0).all()
    close(lse[:B][~empty], want_lse[~empty], s_lse[~empty], L.F32)
    assert torch.isnan(out[B:]).all() and torch.isnan(lse[B:]).all()  # nothing behind the last sequence
    return out, lse


# ------------------------------------------------------------------------------------------------
# Append
# ------------------------------------------------------------------------------------------------

def append_check(P, seq, pos, heads_q, rot, interleaved, pad=0, in_place=False, shift=0, outs=True, stream=None, change=None):
    T, D, dt, g = len(pos), P.D, P.dt, gen(len(pos) + rot)
    cos, sin = L.rotation_tables(max(pos) + 1, rot, device="cuda") if rot else (None, None)
    if rot and shift:
        cos, sin = offset_view(cos, 1), offset_view(sin, 1)

    def token_rows(h):
        t = normal(g, dt, T, h * D + pad)
        t = offset_view(t, shift) if shift else t
        return t, t[:, : h * D].unflatten(-1, (h, D))

    (k_raw, k), (v_raw, v), (q_raw, q) = token_rows(P.heads), token_rows(P.heads), token_rows(max(heads_q, 1))
    if change:
        change(k, v)
    k0, v0, q0 = k.clone(), v.clone(), q.clone()
    k_out, v_out = (k_raw, v_raw) if in_place else (torch.full_like(k_raw, -7.0), torch.full_like(v_raw, -7.0))
    qo_raw = q_raw if in_place else torch.full_like(q_raw, -7.0)
    was = [r.clone() for r in P.raw]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    op = L.KvAppend(P.cache(), P.table, P.seqs, P.width, heads_q=heads_q, cos=cos, sin=sin, max_pos=max(pos) + 1, rot_dim=rot,
                    interleaved=interleaved, k_token=P.heads * D + pad, v_token=P.heads * D + pad,
                    q_token=heads_q * D + pad if heads_q else 0, q_out_token=heads_q * D + pad if heads_q else 0, status=status)
    pos_d = torch.tensor(pos, dtype=torch.int32, device="cuda")
    seq_d = None if seq is None else torch.tensor(seq, dtype=torch.int32, device="cuda")
    op.append(k_raw, v_raw, pos_d, T, seq=seq_d, q=q_raw if heads_q else None, q_out=qo_raw if heads_q else None, stream=stream,
              k_out=k_out if outs else None, v_out=v_out if outs else None)
    torch.cuda.synchronize()
    assert status.item() == 0
    live, dead = torch.nonzero(pos_d >= 0)[:, 0], torch.nonzero(pos_d < 0)[:, 0]
    at, of = pos_d[live].long(), live if seq is None else seq_d[live].long()
    page, slot = P.table.long()[of, at // P.page], at % P.page
    c, s = (cos[at].double()[:, None, :], sin[at].double()[:, None, :]) if rot else (None, None)
    keys = k0[live].double()
    if rot:
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        u, w = keys[..., a].clone(), keys[..., b].clone()
        keys[..., a], keys[..., b] = once(once(u * c) - once(w * s)), once(once(w * c) + once(u * s))
    for which, x, raw, into, given in ((0, keys, was[0], k_out, k0), (1, v0[live].double(), was[1], v_out, v0)):
        n, z, sc = quantised(x, P.group)
        number, word = P.packed(n, z, sc)
        nibbles, words = P.views(raw)
        nibbles[page, slot // 16, :, :, slot % 16] = number
        words[page, slot // 16, :, :, slot % 16] = word
        assert torch.equal(P.raw[which], raw)  # every byte, and every other slot as it was
        got = into[:, : P.heads * D].unflatten(-1, (P.heads, D))
        if outs:
            assert torch.equal(got[live], stand_for(n, z, sc, P.group).to(TORCH[dt]))
            step = sc.repeat_interleave(P.group, -1)[..., :D]
            # A step at most: half of one for the number, half for the zero point (and 2^-18 of it for the quotients).
            assert ((stand_for(n, z, sc, P.group) - x).abs() <= step * (1 + 2.0 ** -17)).all()
        else:
            assert in_place or (into == -7.0).all()
        assert torch.equal(got[dead], (given if in_place else torch.full_like(given, -7.0))[dead])
        if pad and not in_place:
            assert (into[:, P.heads * D:] == -7.0).all()
    if heads_q:
        qo = qo_raw[:, : heads_q * D].unflatten(-1, (heads_q, D))
        want, slack = turned(q0[live], cos[at] if rot else None, sin[at] if rot else None, rot, interleaved)
        close(qo[live], want, slack, dt)
        assert torch.equal(qo[dead], q0[dead] if in_place else torch.full_like(q0[dead], -7.0))


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (80, 32), (64, 0), (66, 34), (33, 2), (2, 2), (256, 256), (48, 48), (1, 0), (200, 24)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_rotations(dt, D, rot, interleaved):
    for group in (32, 64, 128):
        append_check(Pages4(dt, 3, 5, 16, 2, D, group, seed=D), [0] * 40 + [2] * 9, list(range(20, 60)) + list(range(9)), 6, rot, interleaved)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("page,together", [(16, False), (48, True), (64, False)])
@pytest.mark.parametrize("pad,shift,in_place", [(0, 0, True), (8, 0, False), (3, 0, True), (0, 1, False), (3, 1, True)])
def test_append_strides(dt, page, together, pad, shift, in_place):
    P = Pages4(dt, 4, 3, page, 3, 96, 64, seed=pad, together=together)
    append_check(P, [3] * 10 + [1] * 5, list(range(30, 40)) + [0, 1, -1, 2, 41], 3, 96, False, pad, in_place, shift)


@pytest.mark.parametrize("tokens", [1, 2, 31, 700])
def test_append_one_token_per_sequence(tokens):
    P = Pages4(L.BF16, tokens, 3, 16, 2, 64, 32, seed=tokens)
    pos = [(29 * i) % 48 for i in range(tokens)]
    if tokens > 2:
        pos[1] = -3
    append_check(P, None, pos, 4, 64, False)


def test_append_keys_and_values_only():
    append_check(Pages4(L.F16, 2, 4, 16, 2, 64, 64), [1] * 50, list(range(50)), 0, 64, False, outs=False)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_append_ranges(dt):
    """Zeros, one sign alone, the type's smallest and largest numbers, far outliers, and ties between two numbers."""
    def change(k, v):
        big, tiny = torch.finfo(TORCH[dt]).max, torch.finfo(TORCH[dt]).tiny
        v[0], v[1], v[2], v[3], v[4] = 0.0, v[1].abs() + 5, -v[2].abs() - 5, tiny, v[4] * tiny
        v[5, :, 0], v[6] = big * (1 - 2.0 ** -10), torch.where(v[6] > 0, big, -big) * 0.5
        v[7] = torch.arange(v.shape[-1], device="cuda") % 31 / 2 - 4.5  # s = 1: every second one a tie
        k[0], k[1, :, 0] = 0.0, 1000.0
    append_check(Pages4(dt, 1, 2, 16, 2, 128, 64), [0] * 10, list(range(10)), 0, 0, False, change=change)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_append_infinities_and_nans_make_their_group_nan(dt):
    P = Pages4(dt, 1, 1, 16, 1, 96, 32, seed=2)
    g = gen(3)
    k, v = normal(g, dt, 4, 1, 96), normal(g, dt, 4, 1, 96)
    v[0, 0, 3], v[1, 0, 40], v[2, 0, 95] = math.inf, -math.inf, math.nan
    k_out, v_out = torch.empty_like(k), torch.empty_like(v)
    L.KvAppend(P.cache(), P.table, 1, 1).append(k, v, torch.arange(4, dtype=torch.int32, device="cuda"), 4, seq=torch.zeros(4, dtype=torch.int32, device="cuda"),
                                                k_out=k_out, v_out=v_out)
    torch.cuda.synchronize()
    bad = torch.isnan(v_out[:, 0]).unflatten(1, (3, 32))
    assert torch.equal(bad.all(-1), bad.any(-1))
    assert bad.any(-1).nonzero().tolist() == [[0, 0], [1, 1], [2, 2]]
    page = int(P.table[0, 0])
    P.k[page, :4], P.v[page, :4] = k_out.double(), v_out.double()
    q = normal(g, dt, 1, 1, 96)
    out = torch.empty_like(q)
    L.PagedAttention(P.cache(), P.table, 1, 1, 1).decode(q, out, torch.tensor([4], dtype=torch.int32, device="cuda"), 1)
    assert torch.isnan(out).all()
    L.PagedAttention(P.cache(), P.table, 1, 1, 1, window=1).decode(q, out, torch.tensor([4], dtype=torch.int32, device="cuda"), 1)
    assert torch.isfinite(out).all()


def test_append_reports_and_leaves_out_bad_tokens():
    P = Pages4(L.BF16, 2, 4, 16, 1, 64, 64, seed=7)
    was = [r.clone() for r in P.raw]
    k, v, q = normal(gen(1), L.BF16, 5, 1, 64), normal(gen(2), L.BF16, 5, 1, 64), normal(gen(3), L.BF16, 5, 2, 64)
    cos, sin = L.rotation_tables(50, 64, device="cuda")
    for pos, seq, bit, good in [([64, 0, 0, -1, -1], [0, 2, -1, 9, 0], L.KV_BAD_PAGE, []),
                                ([50, 3, 63, -9, -1], [0, 1, 1, 0, 0], L.KV_BAD_POSITION, [1])]:
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        qo, ko = torch.zeros_like(q), torch.zeros_like(k)
        L.KvAppend(P.cache(), P.table, 2, 4, heads_q=2, cos=cos, sin=sin, max_pos=50 if good else 1000, rot_dim=64 if good else 0,
                   status=status).append(k, v, torch.tensor(pos, dtype=torch.int32, device="cuda"), 5, q=q, q_out=qo, k_out=ko,
                                         seq=torch.tensor(seq, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert status.item() == bit
        for t in range(5):
            assert (qo[t] != 0).any() == (ko[t] != 0).any() == (t in good)
        for which in range(2):
            changed = (P.views(P.raw[which])[0] != P.views(was[which])[0]).flatten(5).any(-1).any(3).any(2)  # [page][block][slot]
            assert [[int(P.table[seq[t], pos[t] // 16]), 0, pos[t] % 16] for t in good] == changed.nonzero().tolist()


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("heads,G", [(1, 1), (3, 2), (2, 5), (2, 8), (1, 12), (2, 16), (1, 33)])
def test_attention_head_layouts(dt, heads, G):
    check(Pages4(dt, 5, 20, 16, heads, 64, 64, seed=G), [300, 0, 1, 17, 255], heads * G, dt)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("D", [1, 8, 32, 33, 40, 72, 80, 96, 100, 128, 160, 192, 250, 256])
def test_attention_head_sizes_and_groups(dt, D):
    for group in (32, 64, 128):
        for heads_q in (6, 24):
            check(Pages4(dt, 3, 14, 16, 2, D, group, seed=D), [200, 33, 7], heads_q, dt)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("page,together", [(16, True), (48, False), (128, True)])
def test_attention_pages(dt, page, together):
    check(Pages4(dt, 4, -(-230 // page), page, 2, 64, 32, seed=page, together=together), [230, 65, 64, 63], 8, dt)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("lens", [[5000], [4097, 1], [0, 9000, 3, 2048, 1, 0, 777], [40000], [0], [64] * 40, [(37 * i) % 900 for i in range(200)]])
def test_attention_lengths(dt, lens):
    P = Pages4(dt, len(lens), max(1, -(-max(lens) // 32)), 32, 2, 64, 64, seed=len(lens))
    for scale in (0.0, -0.25):
        first = check(P, lens, 4, dt, scale=scale)
        again = check(P, lens, 4, dt, scale=scale)
        assert all(torch.equal(a[:-1], b[:-1]) for a, b in zip(first, again))  # the same bits every time


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("window", [1, 15, 64, 100, 5000])
def test_attention_window_and_starts(dt, window):
    P = Pages4(dt, 6, 40, 16, 2, 128, 128, seed=window)
    lens = [640, 100, 101, 16, 1, 0]
    check(P, lens, 8, dt, window=window)
    check(P, lens, 8, dt, window=window, starts=[600, 99, 101, -4, 0, 3])


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_attention_scales_of_every_size(dt):
    """Values from 2^-40 to 2^40 of each other, keys that make scores of thousands: scales stay fp32 numbers."""
    P = Pages4(dt, 2, 20, 16, 2, 64, 32, seed=5)
    n, z, s = P.parts[1]
    s = s * torch.exp2(torch.randint(-40, 40, s.shape, device="cuda", generator=gen(6)).double())
    P.v = stand_for(n, z, s, 32)
    number, word = P.packed(n, z, s)
    P.views(P.raw[1])[1].copy_(word.unflatten(1, (-1, 16)).permute(0, 1, 3, 4, 2))
    check(P, [300, 31], 4, L.F32 if dt == L.F16 else dt, plan=None if dt != L.F16 else L.PagedAttention(
        L.KvCache4(P.raw[0], P.raw[1], L.F32, P.num_pages, 16, 2, 64, 32), P.table, 2, 20, 4))
    P = Pages4(dt, 2, 20, 16, 2, 64, 32, seed=5, scale=64.0)
    check(P, [300, 31], 4, dt, scale=0.25)
    check(P, [300, 31], 4, dt, scale=-0.25)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_attention_slots_past_the_end_may_hold_anything(dt):
    P = Pages4(dt, 4, 10, 16, 2, 64, 64, seed=3)
    lens, window = [150, 33, 0, 16], 40
    want = check(P, lens, 8, dt, window=window)
    for b, n in enumerate(lens):
        at = torch.tensor([p for p in range(160) if p >= n or p < n - window], device="cuda")
        page, slot = P.table[b].long()[at // 16], at % 16
        for raw, bits in zip(P.raw, (0x7fffffff, -1)):
            nibbles, words = P.views(raw)
            nibbles[page, 0, :, :, slot] = 255
            words[page, 0, :, :, slot] = bits
    P.table[1, 3:] = -1
    P.table[2, :] = 1 << 30
    got = check(P, lens, 8, dt, window=window)
    assert torch.equal(want[0][:4], got[0][:4]) and torch.equal(want[1][:4], got[1][:4])


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
def test_attention_reports_bad_pages_and_leaves_them_out(dt):
    P = Pages4(dt, 3, 8, 16, 1, 64, 64, seed=6)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, lens = normal(gen(1), dt, 3, 2, 64), torch.tensor([128, -5, 1000], dtype=torch.int32, device="cuda")
    P.table[0, 2], P.table[0, 5] = -1, P.num_pages
    out = torch.empty_like(q)
    L.PagedAttention(P.cache(), P.table, 3, 8, 2, status=status).decode(q, out, lens, 3)
    torch.cuda.synchronize()
    assert status.item() == L.KV_BAD_PAGE
    at = torch.tensor([p for p in range(128) if p // 16 not in (2, 5)], device="cuda")
    rows = P.table[0].long()[at // 16], at % 16
    want = torch.softmax(q[0].double() @ P.k[rows][:, 0].t() / 8.0, -1) @ P.v[rows][:, 0]
    assert (out[0].double() - want).abs().max() < (1e-5 if dt == L.F32 else 2e-2)
    assert torch.equal(out[1], torch.zeros_like(out[1]))
    k, v = (t[:, 0] for t in P.rows(2, 0, 128))
    want = torch.softmax(q[2].double() @ k.t() / 8.0, -1) @ v
    assert (out[2].double() - want).abs().max() < (1e-5 if dt == L.F32 else 2e-2)
    cache = L.KvCache4(None, None, dt, 0, 16, 1, 64, 64)  # a table that points into a cache of no pages
    status.zero_()
    lse = torch.zeros(3, 2, device="cuda")
    L.PagedAttention(cache, P.table, 3, 8, 2, status=status).decode(q, out, lens, 3, lse=lse)
    torch.cuda.synchronize()
    assert status.item() == L.KV_BAD_PAGE and (out == 0).all() and (lse == -math.inf).all()


def test_queries_that_are_not_finite():
    """An infinity in an fp32 query makes infinite scores, of the sign its keys have there; a NaN makes its head NaN."""
    P = Pages4(L.F32, 1, 2, 16, 1, 64, 64, seed=8)
    q = normal(gen(1), L.F32, 1, 3, 64)
    q[0, 1, 5], q[0, 2, 7] = math.inf, math.nan
    out, lse = torch.empty_like(q), torch.empty(1, 3, device="cuda")
    L.PagedAttention(P.cache(), P.table, 1, 2, 3).decode(q, out, torch.tensor([20], dtype=torch.int32, device="cuda"), 1, lse=lse)
    k, v = (t[:, 0] for t in P.rows(0, 0, 20))
    want = torch.softmax(q[0, 0].double() @ k.t() / 8.0, -1) @ v
    assert (out[0, 0].double() - want).abs().max() < 1e-5
    assert torch.isnan(out[0, 2]).all() and not torch.isfinite(lse[0, 1])
    big = torch.full((1, 1, 64), torch.finfo(torch.float32).max, device="cuda")  # not infinite in its first part
    L.PagedAttention(P.cache(), P.table, 1, 2, 1, scale=2.0 ** -130).decode(big, out[:, :1], torch.tensor([20], dtype=torch.int32, device="cuda"), 1)
    want = torch.softmax(big[0, 0].double() @ k.t() * 2.0 ** -130, -1) @ v
    assert (out[0, 0].double() - want).abs().max() < 1e-4


def test_cache_offsets_pass_32_bits():
    """Pages three billion bytes apart are refused; a thousand pages of five million bytes reach past 2^32."""
    page, heads, D = 16, 1, 64
    stride, n = 5_000_000 // 16 * 16, 1000
    buf = torch.empty(stride * n + 4096, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[n - 1, n - 2]], dtype=torch.int32, device="cuda")
    cache = L.KvCache4(buf, buf[2048:], L.BF16, n, page, heads, D, 64, k_page=stride, v_page=stride)
    g = gen(9)
    k, v, q = normal(g, L.BF16, 20, heads, D), normal(g, L.BF16, 20, heads, D), normal(g, L.BF16, 1, 2, D)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    pos, seq = torch.arange(20, dtype=torch.int32, device="cuda"), torch.zeros(20, dtype=torch.int32, device="cuda")
    L.KvAppend(cache, table, 1, 2).append(k, v, pos, 20, seq=seq, k_out=ko, v_out=vo)
    out = torch.empty_like(q)
    L.PagedAttention(cache, table, 1, 2, 2).decode(q, out, torch.tensor([20], dtype=torch.int32, device="cuda"), 1)
    torch.cuda.synchronize()
    want = torch.softmax(q[0].double() @ ko[:, 0].double().t() / 8.0, -1) @ vo[:, 0].double()
    assert (out[0].double() - want).abs().max() < 2e-2


def test_steps_together_in_a_graph():
    """Append and attention of a step, captured and replayed with new inputs, against the same calls one by one."""
    dt, B, H, HK, D = L.BF16, 3, 4, 2, 64
    P = Pages4(dt, B, 20, 16, HK, D, 64, seed=11)
    cos, sin = L.rotation_tables(320, D, device="cuda")
    qkv = normal(gen(1), dt, B, (H + 2 * HK) * D)
    row = qkv.shape[1]
    ap = L.KvAppend(P.cache(), P.table, B, 20, heads_q=H, cos=cos, sin=sin, max_pos=320, rot_dim=D, k_token=row, v_token=row, q_token=row, q_out_token=row)
    slopes = L.distance_slopes(H, device="cuda")
    plan = L.PagedAttention(P.cache(), P.table, B, 20, H, q_token=row, cap=20.0, slopes=slopes)
    pos, lens = torch.tensor([5, 200, 0], dtype=torch.int32, device="cuda"), torch.tensor([6, 201, 1], dtype=torch.int32, device="cuda")
    starts = torch.tensor([2, 100, 0], dtype=torch.int32, device="cuda")
    out = torch.zeros(B, H, D, dtype=TORCH[dt], device="cuda")

    def step(stream):
        ap.append(qkv[:, H * D:], qkv[:, (H + HK) * D:], pos, B, q=qkv, q_out=qkv, stream=stream)
        plan.decode(qkv, out, lens, B, stream=stream, starts=starts)

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
        got = out.clone(), qkv.clone()
        qkv.copy_(new)
        step(None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (out, qkv)))
    assert torch.isfinite(out).all()
    del graph
