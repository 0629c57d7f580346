"""Refusals of the cache in 4 bits and of other attention scores: before any device is touched, so these run without a GPU."""
import pytest

import l2domain_b200 as L

PTR = 0x10000000  # never dereferenced
INVALID, UNSUPPORTED, NO_DEVICE = -1, -7, -3
CACHE = dict(k=PTR, v=PTR, dtype=L.BF16, num_pages=8, page_size=16, heads=2, head_dim=64, group=64)
TABLE = dict(table=PTR, num_seqs=4, table_width=4)
OPS = ("append", "attention")


def call(op, cache=None, table=None, desc=None, **kw):
    c = L.KvCache4(**{**CACHE, **(cache or {})})
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
    (dict(page_size=0), {}, UNSUPPORTED, "multiples of 16"), (dict(page_size=24), {}, UNSUPPORTED, "multiples of 16"),
    (dict(page_size=-16), {}, UNSUPPORTED, "multiples of 16"),
    (dict(group=0), {}, UNSUPPORTED, "groups"), (dict(group=48), {}, UNSUPPORTED, "groups"), (dict(group=256), {}, UNSUPPORTED, "groups"),
    (dict(num_pages=-1), {}, INVALID, "pages"), (dict(num_pages=1 << 31), {}, INVALID, "pages"),
    ({}, dict(num_seqs=-1), INVALID, "table"), ({}, dict(table_width=-1), INVALID, "table"),
    (dict(page_size=1 << 20), dict(table_width=1 << 12), INVALID, "positions"),
    (dict(k_page=1136), {}, INVALID, "apart"), (dict(v_page=1160), {}, INVALID, "apart"), (dict(k_page=-1152), {}, INVALID, "apart"),
    (dict(k_page=1 << 41), {}, INVALID, "too large"), ({}, dict(table_stride=3), INVALID, "strides"),
    (dict(k=None), {}, INVALID, "null"), (dict(v=None), {}, INVALID, "null"), ({}, dict(table=None), INVALID, "null"),
    (dict(k=PTR + 8), {}, INVALID, "aligned"), (dict(v=PTR + 2), {}, INVALID, "aligned"),
    ({}, dict(table=PTR + 2), INVALID, "aligned"), ({}, dict(status=PTR + 1), INVALID, "aligned"),
])
def test_cache_refusals(op, cache, table, status, word):
    with pytest.raises(L.L2DError, match=word) as e:
        call(op, cache, table)
    assert e.value.status == status


@pytest.mark.parametrize("desc,kw,word", [
    (dict(heads_q=-1), {}, "query heads"), (dict(rot_dim=63), {}, "rot_dim"), (dict(rot_dim=66), {}, "rot_dim"),
    ({}, dict(tokens=-1), "tokens"), (dict(k_token=127), {}, "stride"), (dict(q_out_token=1), {}, "stride"),
    (dict(v_token=1 << 58), {}, "too large"), ({}, dict(tokens=5), "without seq"), ({}, dict(k=None), "null"),
    ({}, dict(pos=None), "null"), ({}, dict(q=None), "null"), (dict(cos=None), {}, "null"),
    ({}, dict(k=PTR + 1), "aligned"), ({}, dict(k_out=PTR + 1), "aligned"), ({}, dict(v_out=PTR + 1), "aligned"),
    (dict(max_pos=-1), {}, "max_pos"), (dict(q_token=512), {}, "q_out is q"),
])
def test_append_refusals(desc, kw, word):
    with pytest.raises(L.L2DError, match=word) as e:
        call("append", desc=desc, **kw)
    assert e.value.status == INVALID


def test_append_of_no_tokens_does_nothing():
    call("append", tokens=0)


def test_stored_values_are_of_a_cache_in_4_bits():
    cache = L.KvCache(k=PTR, v=PTR, dtype=L.BF16, num_pages=8, page_size=16, heads=2, head_dim=64)
    with pytest.raises(ValueError, match="4 bits"):
        L.KvAppend(cache, PTR, 4, 4).append(PTR, PTR, PTR, 0, k_out=PTR)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("desc,word", [
    (dict(heads_q=5), "query heads"), (dict(window=-1), "window"), (dict(scale=float("nan")), "scale"), (dict(scale=3e38), "too large"),
    (dict(max_batch=5), "max_batch"), (dict(q_token=255), "stride"),
    (dict(cap=-1.0), "cap"), (dict(cap=float("nan")), "cap"), (dict(cap=float("inf")), "cap"), (dict(cap=3e38), "cap"),
    (dict(cap=1e-39), "cap"), (dict(slopes=PTR + 2), "slopes"),
])
def test_attention_refusals(four, desc, word):
    cache = L.KvCache4(**CACHE) if four else L.KvCache(**{k: v for k, v in CACHE.items() if k != "group"})
    with pytest.raises(L.L2DError, match=word) as e:
        L.PagedAttention(cache, **TABLE, **{**dict(heads_q=4), **desc})
    assert e.value.status == INVALID


def test_page_bytes():
    assert L.kv4_page_bytes(16, 1, 128, 128) == 16 * (64 + 4)
    assert L.kv4_page_bytes(64, 3, 80, 32) == 64 * 3 * (48 + 12)  # rows of whole 16 bytes, a short group
    assert L.lib().l2d_kv4_page_bytes(1, 128, 16, 128, None) == INVALID


def test_calls_without_descriptions():
    import ctypes as C
    lib = L.lib()
    n = C.c_void_p(0)
    for create in (lib.l2d_attn_plan_create_kv4, lib.l2d_attn_plan_create_scored):
        assert create(None, None, None, None) == INVALID
        assert create(None, None, None, C.byref(n)) == INVALID
    cache = L.KvCache4(**CACHE).desc(**TABLE)
    assert lib.l2d_attn_plan_create_kv4(C.byref(cache), None, None, C.byref(n)) == INVALID
    assert lib.l2d_kv4_append(C.byref(cache), None, PTR, PTR, None, None, None, None, PTR, None, 1, None) == INVALID
    assert lib.l2d_attn_decode_from(None, PTR, PTR, None, PTR, None, 1, None) == INVALID


def test_without_a_gpu_the_operators_report_no_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for op in OPS:
        with pytest.raises(L.L2DError) as e:
            call(op)
        assert e.value.status == NO_DEVICE


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("side", ["k_page", "v_page"])
@pytest.mark.parametrize("bytes_apart", [(1 << 31) + 16, 3_000_000_000 // 16 * 16])
def test_pages_more_than_2_31_bytes_apart_are_refused(op, side, bytes_apart):
    with pytest.raises(L.L2DError, match="too large") as e:
        call(op, {side: bytes_apart})
    assert e.value.status == INVALID
