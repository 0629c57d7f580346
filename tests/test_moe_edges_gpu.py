"""The mixture-of-experts layer on the GPU where memory, ranges and precision end (tolerances: test_moe_gpu.py, unless a test
derives its own)."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import l2domain_b200 as L  # noqa: E402
from l2domain_b200 import decode  # noqa: E402
from test_decode_ops_gpu import TORCH, close, gpu, offset_view  # noqa: E402,F401
from test_moe_gpu import Layer, check  # noqa: E402


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("name", ["router", "gate", "up", "down"])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_one_matrix_alone_off_its_boundary(dt, name, shift):
    """Every other matrix is on 16 bytes, and the last step of each product is short: by runs without an element too."""
    for H, F in ((72, 40), (32, 104), (1000, 88)):
        layer = Layer(dt, H, F, 4, 2, seed=H)
        moved = offset_view(getattr(layer, name + "_raw"), shift)
        setattr(layer, name + "_raw", moved)
        setattr(layer, name, moved)
        for T in (1, 20):
            check(layer, T)


@pytest.mark.parametrize("dt", [L.F16, L.BF16])
@pytest.mark.parametrize("H", [72, 73])
def test_odd_rows_beside_even_ones(dt, H):
    """Rows of each matrix in turn begin in the middle of a word, `down` also off every boundary."""
    for pads in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0)):
        layer = Layer(dt, H, 72, 3, 2, seed=H)
        for name, pad in zip(("gate", "up", "down"), pads):
            m = getattr(layer, name)
            wide = torch.zeros(*m.shape[:-1], m.shape[-1] + pad, dtype=m.dtype, device="cuda")
            wide[..., : m.shape[-1]] = m
            if name == "down":
                wide = offset_view(wide, 1)
            setattr(layer, name + "_raw", wide)
            setattr(layer, name, wide[..., : m.shape[-1]])
        check(layer, 5)


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_an_infinite_inner_value_keeps_the_sign_of_its_outputs(sign):
    """fp16: one inner value is infinite and others are beyond 65504 and pull the other way: the outputs are infinite still."""
    H, F = 16, 24
    layer = Layer(L.F16, H, F, 1, 1, seed=11)
    layer.gate[:], layer.up[:] = 0.0, 0.0
    layer.gate[0, :, 0] = 1.0     # gates of 500
    layer.up[0, :, 1] = 500.0     # ups of 2000, so inner values of 10^6 ..
    layer.up[0, 3, 2] = math.inf  # .. and row 3's is infinite
    layer.down[:] = -sign
    layer.down[0, :, 3] = sign
    x = torch.zeros(1, H, dtype=torch.float16, device="cuda")
    x[0, 0], x[0, 1], x[0, 2] = 500.0, 4.0, 1.0
    y = torch.zeros_like(x)
    layer.plan(1).forward(x, y, 1)
    torch.cuda.synchronize()
    assert (y == sign * math.inf).all()


@pytest.mark.parametrize("dt", [L.F32, L.F16, L.BF16])
@pytest.mark.parametrize("E,top", [(1, 1), (8, 2), (32, 32), (100, 5), (512, 16)])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("spread", [0.05, 1.0, 8.0])
def test_routing_weights_are_rounded_once(dt, E, top, normalize, spread):
    """Weights are taken in 64 bits, of sums in 64 bits, and rounded to fp32: half a unit in the last place is 2^-24 of a
    weight; the sums of 64 products, some 80 in all at the largest spread, are off by 64 * 80 * 2^-53 at most on either side, which
    with exp and the quotient is less than 2^-38 of a weight.  Below 2^-126 a unit is 2^-149."""
    layer = Layer(dt, 64, 8, E, top, seed=E)
    layer.router[:] = (layer.router.float() * spread).to(TORCH[dt])
    x = layer.tokens(40)
    y = torch.empty_like(x)
    w = torch.full((40, top), math.nan, device="cuda")
    layer.plan(40, normalize).forward(x, y, 40, weights=w)
    torch.cuda.synchronize()
    _, _, _, want = layer.exact(x, normalize)
    assert ((w.double() - want).abs() <= (2.0 ** -24 + 2.0 ** -38) * want + 2.0 ** -149).all()


def test_experts_of_the_decoding_layer_may_be_strided():
    """Rows and experts of views, and sizes of one whose strides say nothing."""
    for E, F, H, top in ((3, 24, 40, 2), (1, 8, 16, 1), (2, 1, 8, 1), (2, 8, 1, 2)):
        layer = Layer(L.BF16, H, F, E, top, seed=F)
        wide = torch.zeros(E, F, 2, H + 3, dtype=torch.bfloat16, device="cuda")
        wide[:, :, 0, :H], wide[:, :, 1, :H] = layer.gate, layer.up
        router = torch.zeros(E, 2 * H, dtype=torch.bfloat16, device="cuda")[:, H:]
        router.copy_(layer.router)
        down = layer.down.as_strided((E, H, F), tuple(s if n > 1 else 5 for n, s in zip((E, H, F), layer.down.stride())))
        moe = decode.DecodeExperts(router, wide[:, :, 0, :H], wide[:, :, 1, :H], down, top, 4)
        x = layer.tokens(4)
        y = torch.empty_like(x)
        moe.step(x, y)
        torch.cuda.synchronize()
        want, slack, ids, _ = layer.exact(x, True)
        assert torch.equal(moe.ids.long(), ids)
        close(y, want, slack, L.BF16)


def test_inner_values_of_bf16_keep_what_fp32_holds():
    """Outputs that are differences of two nearly equal inner values.  Their sums are one exact product each; exp is off by two
    units (2^-22), the three operations after it by 2^-24 each: 14 * 2^-24 of the larger for two.  The difference: three parts of each,
    in six instructions at most, that cut two operands off at the last place of the largest (2^-23): 24 * 2^-24."""
    H, F = 2048, 4096
    layer = Layer(L.BF16, H, F, 1, 1, seed=12)
    g = layer.g
    layer.gate[:], layer.up[:], layer.down[:] = 0.0, 0.0, 0.0
    layer.gate[0, :, 0] = torch.empty(F, device="cuda").uniform_(1.0, 2.0, generator=g).bfloat16()
    layer.up[0, :, 1] = torch.empty(F, device="cuda").uniform_(1.0, 2.0, generator=g).bfloat16()
    x = torch.zeros(1, H, dtype=torch.bfloat16, device="cuda")
    x[0, 0], x[0, 1] = 1.171875, 1.3203125
    a, b = (m[0].double() @ x[0].double() for m in (layer.gate, layer.up))
    h = a * torch.sigmoid(a) * b
    order = torch.sort(h)[1].view(H, 2)
    rows = torch.arange(H, device="cuda")
    layer.down[0, rows, order[:, 1]], layer.down[0, rows, order[:, 0]] = 1.0, -1.0
    y = torch.empty_like(x)
    layer.plan(1).forward(x, y, 1)
    torch.cuda.synchronize()
    want = h[order[:, 1]] - h[order[:, 0]]
    assert want.abs().mean() < 2.0 ** -9 * h.mean()
    close(y[0], want, 38 * 2.0 ** -24 * h[order].amax(1), L.BF16)


@pytest.mark.parametrize("dt", [L.F16, L.BF16])
def test_an_odd_inner_value_is_its_slots_alone(dt):
    """A token whose inner values are not finite beside others of the same expert, in one call and in the next."""
    layer = Layer(dt, 64, 72, 2, 1, seed=13)
    x = layer.tokens(20)
    clean = check(layer, 20, x=x)[0]
    plan, bad = layer.plan(20), x.clone()
    bad[3], bad[11] = math.inf, math.nan
    y = torch.empty_like(x)
    plan.forward(bad, y, 20)
    torch.cuda.synchronize()
    rest = [t for t in range(20) if t not in (3, 11)]
    assert torch.equal(y[rest], clean[rest]) and not torch.isfinite(y[[3, 11]]).any()
    assert torch.equal(check(layer, 20, x=x, plan=plan)[0], clean)


def test_small_inner_values_of_fp16_beside_a_large_one():
    """Inner values are cut into two fp16 numbers relative to the largest, M = 2^14 .. 2^15 then: the second is off by 2^-25 where
    it is subnormal, 2^-39 of M.  Beside that an output is off by silu's seven roundings of 2^-24 (an exp of two units and three
    operations; sums are one exact product each), down times."""
    H, F = 64, 256
    layer = Layer(L.F16, H, F, 1, 1, seed=14)
    layer.gate[:], layer.up[:], layer.down[:] = 0.0, 0.0, 0.0
    layer.gate[0, :, 0] = torch.empty(F, device="cuda").uniform_(1.0, 2.0, generator=layer.g).half()
    layer.up[0, :, 1] = torch.exp2(-torch.empty(F, device="cuda").uniform_(0.0, 14.0, generator=layer.g)).half()
    layer.up[0, 0, 1], layer.up[0, 0, 2] = 0.0, 32768.0  # the largest
    layer.down[0, :, :H] = 0.0
    rows, at = torch.arange(H, device="cuda"), torch.arange(1, H + 1, device="cuda") * 3
    layer.down[0, rows, at] = 32768.0
    x = torch.zeros(1, H, dtype=torch.float16, device="cuda")
    x[0, 0], x[0, 1], x[0, 2] = 1.0, 2.0 ** -13, 1.0
    y = torch.empty_like(x)
    layer.plan(1).forward(x, y, 1)
    torch.cuda.synchronize()
    a, b = (m[0].double() @ x[0].double() for m in (layer.gate, layer.up))
    h = a * torch.sigmoid(a) * b
    assert (h[1:] < 2.0 ** -27 * h[0]).all() and (h[at] < 2.0 ** -30 * h[0]).any()
    close(y[0], 32768.0 * h[at], 32768.0 * (2.0 ** -39 * h[0] + (2.0 ** -22 + 7 * 2.0 ** -24) * h[at]), L.F16)
