"""The mixture-of-experts layer on the GPU against its definition in 64 bits.

Tolerances, per element, from rounding alone (u = 2^-24; sums in any order, a matrix instruction may truncate where it adds,
which costs twice a rounding): a sum of n terms is off by 2u (160 + n / 16) S, S the sum of the terms' absolute
values; silu has a slope of at most 1.1 and its value, times up, four roundings and two units of exp; what meets the down
product is held to 2^-16 (bf16: two numbers of 8 bits), or to 2^-22 and 2^-38 of the slot's largest (fp16), or exactly.  A weight is
a quotient of fp32 numbers: expf is off by two units (2^-22), its argument's second half by a rounding (2^-24), above and below;
the sum below has up to 16 + 5 additions of positive numbers (21 * 2^-24), the quotient a rounding: 2^-21 + 24 * 2^-24 <
2^-19 of itself.  The sum over a token's choices is off by one rounding each.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import l2domain_b200 as L  # noqa: E402
from test_decode_ops_gpu import TORCH, U, close, gen, gpu, offset_view  # noqa: E402,F401

HELD = {L.F32: (0.0, 0.0), L.F16: (2.0 ** -22, 2.0 ** -38), L.BF16: (2.0 ** -16, 0.0)}


class Layer:
    def __init__(self, dt, H, F, E, top, seed=0, pad=0, shift=0, together=False, scale=1.0):
        g = gen(seed)
        self.dt, self.H, self.F, self.E, self.top, self.g = dt, H, F, E, top, g

        def normal(*shape, s):
            t = (torch.empty(*shape[:-1], shape[-1] + pad, device="cuda").normal_(generator=g) * s).to(TORCH[dt])
            return offset_view(t, shift) if shift else t

        self.router_raw, self.down_raw = normal(E, H, s=2.0 * H ** -0.5), normal(E, H, F, s=scale * F ** -0.5)
        if together:  # gate and up row by row in one buffer
            both = normal(E, F, 2, H, s=scale * H ** -0.5)
            self.gate_raw, self.up_raw = both[:, :, 0], both[:, :, 1]
        else:
            self.gate_raw, self.up_raw = (normal(E, F, H, s=scale * H ** -0.5) for _ in range(2))
        self.router, self.gate, self.up, self.down = (t[..., :n] for t, n in zip((self.router_raw, self.gate_raw, self.up_raw, self.down_raw), (H, H, H, F)))

    def plan(self, max_tokens, normalize=True, **kw):
        return L.MoeLayer(self.router_raw, self.gate_raw, self.up_raw, self.down_raw, self.H, self.F, self.E, self.top, max_tokens, self.dt, normalize,
                          router_row=self.router_raw.stride(0), gate_row=self.gate_raw.stride(1), up_row=self.up_raw.stride(1),
                          down_row=self.down_raw.stride(1), gate_expert=self.gate_raw.stride(0), up_expert=self.up_raw.stride(0),
                          down_expert=self.down_raw.stride(0), **kw)

    def tokens(self, T, scale=1.0):
        return (torch.empty(T, self.H, device="cuda").normal_(generator=self.g) * scale).to(TORCH[self.dt])

    def exact(self, x, normalize):
        """(y, slack, ids, weights) in 64 bits."""
        T = x.shape[0]
        x = x.double()
        logits = x @ self.router.double().t()
        ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, : self.top]
        w = torch.softmax(logits, 1).gather(1, ids)
        if normalize:
            w = w / w.sum(1, keepdim=True)
        y, slack = torch.zeros_like(x), torch.zeros_like(x)
        held, least = HELD[self.dt]
        grow_up, grow_down = 2 * U * (160 + self.H / 16), 2 * U * (160 + self.F / 16)
        for e in range(self.E):
            t, k = torch.nonzero(ids == e, as_tuple=True)
            if not len(t):
                continue
            gate, up, down = (m[e].double() for m in (self.gate, self.up, self.down))
            a, b = x[t] @ gate.t(), x[t] @ up.t()
            da, db = grow_up * (x[t].abs() @ gate.abs().t()), grow_up * (x[t].abs() @ up.abs().t())
            silu = a * torch.sigmoid(a)
            h = silu * b
            dh = 1.1 * da * (b.abs() + db) + silu.abs() * db + 8 * U * h.abs() + held * h.abs() + least * h.abs().amax(1, keepdim=True)
            part = h @ down.t()
            dpart = dh @ down.abs().t() + grow_down * (h.abs() @ down.abs().t())
            weight = w[t, k][:, None]
            y.index_add_(0, t, weight * part)
            slack.index_add_(0, t, weight * (dpart + (2.0 ** -19 + self.top * 2 * U) * part.abs()))
        return y, slack, ids, w


def check(layer, T, normalize=True, x=None, plan=None, stream=None, y_pad=0):
    x = layer.tokens(T) if x is None else x
    plan = plan or layer.plan(T, normalize, y_token=layer.H + y_pad)
    y = torch.full((T + 1, layer.H + y_pad), math.nan, dtype=TORCH[layer.dt], device="cuda")
    ids = torch.full((T + 1, layer.top), -5, dtype=torch.int32, device="cuda")
    w = torch.full((T + 1, layer.top), math.nan, device="cuda")
    plan.forward(x, y, T, ids=ids, weights=w, stream=stream)
    torch.cuda.synchronize()
    want, slack, want_ids, want_w = layer.exact(x, normalize)
    assert torch.equal(ids[:T].long(), want_ids)
    close(w[:T], want_w, 2.0 ** -19 * want_w, L.F32)
    close(y[:T, : layer.H], want, slack, layer.dt)
    assert torch.isnan(y[T:]).all() and torch.isnan(y[:, layer.H:]).all() and (ids[T:] == -5).all() and torch.isnan(w[T:]).all()
    return y[:T, : layer.H].clone(), ids[:T].clone(), w[:T].clone()


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("H,F", [(1, 1), (8, 8), (64, 32), (33, 7), (128, 200), (1000, 72), (257, 129), (40, 513), (2048, 96), (96, 2050)])
def test_sizes(dt, H, F):
    for T in (1, 5):
        check(Layer(dt, H, F, 6, 2, seed=H), T)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 16, 17, 32, 33, 70, 200])
def test_tokens(dt, T):
    check(Layer(dt, 256, 136, 8, 2, seed=T), T, normalize=T % 2 == 0)


@pytest.mark.parametrize("dt", [L.F32, L.BF16])
@pytest.mark.parametrize("E,top", [(1, 1), (2, 2), (5, 5), (33, 32), (60, 6), (129, 8), (512, 3), (300, 1)])
@pytest.mark.parametrize("normalize", [False, True])
def test_experts(dt, E, top, normalize):
    check(Layer(dt, 96, 40, E, top, seed=E), 11, normalize)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("pad,shift,together", [(8, 0, False), (2, 0, False), (1, 0, False), (0, 1, False), (0, 2, True), (3, 0, True), (0, 0, True)])
def test_strides_and_alignment(dt, pad, shift, together):
    check(Layer(dt, 136, 88, 4, 2, seed=pad, pad=pad, shift=shift, together=together), 6, y_pad=pad)
    layer = Layer(dt, 136, 88, 4, 2, seed=pad)  # only tokens off their boundaries
    x = layer.tokens(6)
    wide = torch.zeros(6, 136 + pad, dtype=x.dtype, device="cuda")
    wide[:, :136] = x
    moved = offset_view(wide, shift)
    check(layer, 6, x=x, plan=None)
    y = torch.empty_like(x)
    layer.plan(6, x_token=136 + pad).forward(moved, y, 6)
    want, slack, _, _ = layer.exact(x, True)
    close(y, want, slack, dt)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_long_rows_and_many_items(dt):
    check(Layer(dt, 8200, 48, 3, 2, seed=1), 3)
    check(Layer(dt, 64, 9000, 3, 2, seed=2), 3)
    check(Layer(dt, 1024, 1024, 16, 4, seed=3), 64)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_the_same_bits_whoever_comes_along(dt):
    """A token's result does not depend on the others, nor on the call."""
    layer = Layer(dt, 320, 200, 12, 3, seed=4)
    x = layer.tokens(40)
    y, ids, w = check(layer, 40, x=x)
    plan = layer.plan(40)
    for _ in range(2):
        again = check(layer, 40, x=x, plan=plan)
        assert torch.equal(again[0], y) and torch.equal(again[1], ids) and torch.equal(again[2], w)
    few = check(layer, 3, x=x[:3].contiguous(), plan=plan)
    assert torch.equal(few[1], ids[:3]) and torch.equal(few[2], w[:3])
    back = check(layer, 40, x=x.flip(0).contiguous(), plan=plan)
    assert torch.equal(back[0].flip(0), y)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_one_expert_for_all_and_ties(dt):
    """All tokens on the same experts; equal router rows: the lower expert wins."""
    layer = Layer(dt, 64, 48, 10, 3, seed=5)
    layer.router[:] = 0
    _, ids, w = check(layer, 50)
    assert (ids == torch.arange(3, device="cuda")).all() and ((w - 1 / 3).abs() < 1e-6).all()
    layer.router[7] = layer.router[4] = layer.router[9] = 1.0
    x = layer.tokens(50).abs()
    _, ids, _ = check(layer, 50, x=x)
    assert (ids == torch.tensor([4, 7, 9], device="cuda")).all()


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("scale", [2.0 ** -12, 2.0 ** 4])
def test_small_and_large_inner_values(dt, scale):
    """Inner values far below and above those of fp16's range (with a scale of 16, products of 2^20 and more)."""
    layer = Layer(dt, 256, 128, 4, 2, seed=6, scale=scale)
    x = layer.tokens(9, 64.0 if scale > 1 else 0.01)
    if dt == L.F16 and scale > 1:
        layer.down_raw *= 2.0 ** -14  # keeps y in the type's range
    check(layer, 9, x=x)


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
def test_infinities_and_nans_stay_with_their_token(dt):
    layer = Layer(dt, 128, 64, 5, 2, seed=7)
    x = layer.tokens(12)
    clean = check(layer, 12, x=x)[0]
    bad = x.clone()
    bad[3, 5], bad[7, 9] = math.nan, math.inf
    y, ids, w = torch.empty_like(x), torch.empty(12, 2, dtype=torch.int32, device="cuda"), torch.empty(12, 2, device="cuda")
    layer.plan(12).forward(bad, y, 12, ids=ids, weights=w)
    torch.cuda.synchronize()
    rest = [t for t in range(12) if t not in (3, 7)]
    assert torch.equal(y[rest], clean[rest])
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[7]).any()
    assert ((ids >= 0) & (ids < 5)).all() and (ids[:, 0] != ids[:, 1]).all()


def test_offsets_pass_32_bits():
    """Experts of two billion elements apart."""
    H, F, E = 64, 32, 3
    stride = (1 << 30) + 64
    buf = torch.empty(stride * 2 + 3 * F * H, dtype=torch.float16, device="cuda")
    layer = Layer(L.F16, H, F, E, 3, seed=8)
    views = []
    for i, m in enumerate((layer.gate, layer.up, layer.down)):
        flat = buf[i * F * H:]
        for e in range(E):
            flat[e * stride: e * stride + F * H] = m[e].reshape(-1)
        views.append(flat)
    plan = L.MoeLayer(layer.router, *views, H, F, E, 3, 4, L.F16, gate_expert=stride, up_expert=stride, down_expert=stride)
    check(layer, 4, plan=plan)


def test_layer_follows_its_stream_and_replays_in_a_graph():
    layer = Layer(L.BF16, 512, 256, 16, 4, seed=9)
    plan, x = layer.plan(16), layer.tokens(16)
    y = torch.zeros_like(x)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    first = x.clone()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            big = big @ big * 1e-3
        x.mul_(2.0)
        plan.forward(x, y, 16, stream=s)
        y2 = y * 1.0
    s.synchronize()
    want, slack, _, _ = layer.exact(x, True)
    close(y2, want, slack, L.BF16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.forward(x, y, 16, stream=torch.cuda.current_stream())
        plan.forward(y, x, 16, stream=torch.cuda.current_stream())
    for n in range(3):
        new = first * (n + 1)
        x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = x.clone(), y.clone()
        x.copy_(new)
        plan.forward(x, y, 16)
        plan.forward(y, x, 16)
        torch.cuda.synchronize()
        assert torch.equal(got[0], x) and torch.equal(got[1], y)
    del graph
