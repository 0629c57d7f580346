"""Refusals of the decoding operators (l2d_q4_gemv, l2d_kv_append, l2d_attn_*): every bad argument the host
can see comes back as a status with a message, before any device is touched, so these run without a GPU."""
import ctypes as C

import pytest

import l2domain_b200 as L

PTR = 0x10000000  # never dereferenced: every call here is refused, or has nothing to do
INVALID, UNSUPPORTED, NO_DEVICE = -1, -7, -3


def q4(x=PTR, y=PTR + (1 << 20), vectors=1, stride_x=0, stride_y=0, **kw):
    f = dict(weights=PTR, scales=PTR, M=16, N=256, group=128, dtype_x=L.F16)
    f.update(kw)
    L.Q4Matrix(**f).gemv(x, y, vectors=vectors, stride_x=stride_x, stride_y=stride_y)


@pytest.mark.parametrize("bad,word", [
    (dict(M=-1), "M = -1"), (dict(N=-5), "N = -5"), (dict(M=1 << 31), "2^31"), (dict(N=1 << 31), "2^31"),
    (dict(group=0), "group"), (dict(group=16), "group"), (dict(group=96), "group"), (dict(group=-128), "group"),
    (dict(dtype_x=3), "dtype"), (dict(dtype_y=-1), "dtype"), (dict(dtype_s=9), "dtype"),
    (dict(ldw=127), "ldw"), (dict(lds=1), "lds"), (dict(vectors=-1), "vectors"),
    (dict(vectors=2, stride_x=255), "overlap"), (dict(vectors=2, stride_y=15), "overlap"),
    (dict(ldw=1 << 59), "too large"), (dict(vectors=4, stride_x=1 << 60), "too large"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(weights=None), "null"), (dict(scales=None), "null"),
    (dict(x=PTR + 1), "aligned"), (dict(y=PTR + 1), "aligned"), (dict(scales=PTR + 1), "aligned"),
])
def test_q4_refusals(bad, word):
    with pytest.raises(L.L2DError, match=word.replace("^", r"\^")) as e:
        q4(**bad)
    assert e.value.status == INVALID


def test_q4_null_descriptor_and_empty_calls():
    assert L.lib().l2d_q4_gemv(None, PTR, 0, PTR, 0, 1, None) == INVALID
    q4(M=0)
    q4(vectors=0)


CACHE = dict(k=PTR, v=PTR, dtype=L.BF16, num_pages=8, page_size=16, heads=2, head_dim=64)
TABLE = dict(table=PTR, num_seqs=4, table_width=4)
OPS = ("append", "attention")


def call(op, cache=None, table=None, desc=None, **kw):
    c = L.KvCache(**{**CACHE, **(cache or {})})
    t = {**TABLE, **(table or {})}
    if op == "append":
        d = {**dict(heads_q=4, cos=PTR, sin=PTR, max_pos=64, rot_dim=64), **(desc or {})}
        a = {**dict(k=PTR, v=PTR, pos=PTR, tokens=4, q=PTR, q_out=PTR), **kw}
        L.KvAppend(c, **t, **d).append(**a)
    else:
        L.PagedAttention(c, **t, **{**dict(heads_q=4), **(desc or {})})


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("cache,table,status,word", [
    (dict(dtype=5), {}, INVALID, "dtype"), (dict(heads=0), {}, INVALID, "heads"), (dict(heads=65536), {}, INVALID, "heads"),
    (dict(head_dim=0), {}, UNSUPPORTED, "head_dim"), (dict(head_dim=257), {}, UNSUPPORTED, "head_dim"),
    (dict(page_size=0), {}, INVALID, "pages"), (dict(num_pages=-1), {}, INVALID, "pages"),
    (dict(num_pages=1 << 31), {}, INVALID, "pages"),
    ({}, dict(num_seqs=-1), INVALID, "table"), ({}, dict(table_width=-1), INVALID, "table"),
    (dict(page_size=1 << 20), dict(table_width=1 << 12), INVALID, "positions"),
    (dict(k_strides=(2048, 63, 64)), {}, INVALID, "strides"), (dict(v_strides=(-1, 128, 64)), {}, INVALID, "strides"),
    ({}, dict(table_stride=3), INVALID, "strides"), (dict(k_strides=(1 << 41, 128, 64)), {}, INVALID, "too large"),
    (dict(k=None), {}, INVALID, "null"), (dict(v=None), {}, INVALID, "null"), ({}, dict(table=None), INVALID, "null"),
    (dict(num_pages=0), dict(table=None), INVALID, "null"),
    (dict(k=PTR + 1), {}, INVALID, "aligned"), (dict(v=PTR + 1), {}, INVALID, "aligned"),
    ({}, dict(table=PTR + 2), INVALID, "aligned"), ({}, dict(status=PTR + 1), INVALID, "aligned"),
])
def test_cache_refusals(op, cache, table, status, word):
    with pytest.raises(L.L2DError, match=word) as e:
        call(op, cache, table)
    assert e.value.status == status


@pytest.mark.parametrize("desc,kw,word", [
    (dict(heads_q=-1), {}, "query heads"), (dict(rot_dim=-2), {}, "rot_dim"), (dict(rot_dim=63), {}, "rot_dim"),
    (dict(rot_dim=66), {}, "rot_dim"), ({}, dict(tokens=-1), "tokens"), (dict(k_token=127), {}, "stride"),
    (dict(q_token=255), {}, "stride"), (dict(q_out_token=1), {}, "stride"), (dict(v_token=1 << 58), {}, "too large"),
    ({}, dict(tokens=5), "without seq"), ({}, dict(k=None), "null"), ({}, dict(v=None), "null"), ({}, dict(pos=None), "null"),
    ({}, dict(q=None), "null"), ({}, dict(q_out=None), "null"), (dict(cos=None), {}, "null"), (dict(sin=None), {}, "null"),
    ({}, dict(k=PTR + 1), "aligned"), ({}, dict(q_out=PTR + 1), "aligned"), ({}, dict(pos=PTR + 2), "aligned"),
    (dict(cos=PTR + 2), {}, "aligned"), (dict(max_pos=-1), {}, "max_pos"),
])
def test_append_refusals(desc, kw, word):
    with pytest.raises(L.L2DError, match=word) as e:
        call("append", desc=desc, **kw)
    assert e.value.status == INVALID


def test_append_of_no_tokens_does_nothing():
    call("append", tokens=0)


@pytest.mark.parametrize("desc,word", [
    (dict(heads_q=0), "query heads"), (dict(heads_q=5), "query heads"), (dict(window=-1), "window"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(max_batch=5), "max_batch"),
    (dict(max_batch=-1), "max_batch"), (dict(q_token=255), "stride"), (dict(out_token=255), "stride"),
    (dict(q_token=1 << 41), "too large"),
])
def test_attention_refusals(desc, word):
    with pytest.raises(L.L2DError, match=word) as e:
        call("attention", desc=desc)
    assert e.value.status == INVALID


def test_attention_calls_without_a_plan():
    lib = L.lib()
    assert lib.l2d_attn_decode(None, PTR, PTR, None, PTR, 1, None) == INVALID
    assert lib.l2d_attn_plan_create(None, None, None) == INVALID
    assert lib.l2d_attn_plan_create(None, C.byref(L.AttnDesc(heads_q=1)), C.byref(C.c_void_p(0))) == INVALID
    assert lib.l2d_attn_plan_destroy(None) == 0


def test_without_a_gpu_the_operators_report_no_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for f in (q4, lambda: call("append"), lambda: call("attention")):
        with pytest.raises(L.L2DError) as e:
            f()
        assert e.value.status == NO_DEVICE


def test_rotation_tables_hold_rounded_angles():
    import numpy as np
    cos, sin = L.rotation_tables(4097, 8, theta=100.0, stretch=4.0)
    p, i = 4096, 3
    angle = np.float64(p) * 100.0 ** (-2.0 * i / 8) / 4.0
    assert cos.shape == sin.shape == (4097, 4)
    assert abs(float(cos[p, i]) - np.cos(angle)) < 1e-7 and abs(float(sin[p, i]) - np.sin(angle)) < 1e-7
