"""Refusals of the mixture-of-experts layer: before any device is touched, so these run without a GPU."""
import ctypes as C

import pytest

import l2domain_b200 as L

PTR = 0x10000000  # never dereferenced
INVALID, UNSUPPORTED, NO_DEVICE = -1, -7, -3


def layer(**kw):
    return L.MoeLayer(**{**dict(router=PTR, gate=PTR, up=PTR, down=PTR, hidden=64, inner=32, experts=4, top=2, max_tokens=8), **kw})


@pytest.mark.parametrize("bad,status,word", [
    (dict(dtype=3), INVALID, "dtype"), (dict(hidden=0), INVALID, "hidden"), (dict(inner=-1), INVALID, "inner"), (dict(hidden=1 << 25), INVALID, "hidden"),
    (dict(experts=0), UNSUPPORTED, "experts"), (dict(experts=513), UNSUPPORTED, "experts"), (dict(top=0), UNSUPPORTED, "top"),
    (dict(top=5), UNSUPPORTED, "top"), (dict(experts=64, top=33), UNSUPPORTED, "top"), (dict(max_tokens=0), INVALID, "max_tokens"),
    (dict(max_tokens=65536), INVALID, "max_tokens"), (dict(router_row=63), INVALID, "stride"), (dict(down_row=31), INVALID, "stride"),
    (dict(x_token=1), INVALID, "stride"), (dict(y_token=-64), INVALID, "stride"), (dict(gate_expert=63), INVALID, "experts' strides"),
    (dict(down_expert=-1), INVALID, "experts' strides"), (dict(gate_row=1 << 33), INVALID, "too large"), (dict(up_expert=1 << 50), INVALID, "too large"),
    (dict(router=None), INVALID, "null"), (dict(gate=None), INVALID, "null"), (dict(up=None), INVALID, "null"), (dict(down=None), INVALID, "null"),
    (dict(gate=PTR + 1), INVALID, "aligned"), (dict(down=PTR + 2, dtype=L.F32), INVALID, "aligned"),
    (dict(hidden=1 << 24, inner=1, experts=512, top=32, max_tokens=65535), INVALID, "2\\^31"),
])
def test_refusals(bad, status, word):
    with pytest.raises(L.L2DError, match=word) as e:
        layer(**bad)
    assert e.value.status == status


def test_calls_without_a_plan():
    lib = L.lib()
    assert lib.l2d_moe_plan_create(None, None) == INVALID
    assert lib.l2d_moe_plan_create(None, C.byref(C.c_void_p(0))) == INVALID
    assert lib.l2d_moe_forward(None, PTR, PTR, None, None, 1, None) == INVALID
    assert lib.l2d_moe_plan_destroy(None) == 0


def test_without_a_gpu_the_layer_reports_no_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(L.L2DError) as e:
        layer()
    assert e.value.status == NO_DEVICE


@pytest.mark.gpu
def test_refusals_of_a_call():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    w = torch.zeros(4 * 64 * 32, dtype=torch.bfloat16, device="cuda")
    plan, x = layer(router=w, gate=w, up=w, down=w), torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    for args, word in (((x, x, -1), "tokens"), ((x, x, 9), "tokens"), ((None, x, 1), "null"), ((x, None, 1), "null"),
                       ((x.data_ptr() + 1, x, 1), "aligned")):
        with pytest.raises(L.L2DError, match=word):
            plan.forward(*args)
    with pytest.raises(L.L2DError, match="aligned"):
        plan.forward(x, x, 1, ids=x.data_ptr() + 2)
    plan.forward(x, x, 0)
