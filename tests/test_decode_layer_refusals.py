"""What the decoding layer's classes refuse of the tensors they are given: before any device is touched, so these run without a GPU."""
import pytest

torch = pytest.importorskip("torch")

import l2domain_b200 as L  # noqa: E402
from l2domain_b200 import decode  # noqa: E402


def experts(dtype=torch.bfloat16, **kw):
    E, F, H = 4, 8, 16
    w = dict(router=torch.zeros(E, H, dtype=dtype), gate=torch.zeros(E, F, H, dtype=dtype), up=torch.zeros(E, F, H, dtype=dtype),
             down=torch.zeros(E, H, F, dtype=dtype))
    w.update(kw)
    return decode.DecodeExperts(**w, top=2, batch=3)


@pytest.mark.parametrize("bad,word", [
    (dict(router=torch.zeros(4, 16)), "router is torch.float32"), (dict(up=torch.zeros(4, 8, 16)), "up is torch.float32"),
    (dict(down=torch.zeros(4, 16, 8, dtype=torch.float16)), "down is torch.float16"), (dict(gate=torch.zeros(4, 8, 16, dtype=torch.float64)), "gate is"),
    (dict(gate=torch.zeros(8, 16, dtype=torch.bfloat16)), "gate is"), (dict(gate=torch.zeros(4, 8, 16)), "router is torch.bfloat16"),
    (dict(router=torch.zeros(3, 16, dtype=torch.bfloat16)), "router has the shape"), (dict(router=torch.zeros(16, 4, dtype=torch.bfloat16)), "router has the shape"),
    (dict(up=torch.zeros(4, 16, 8, dtype=torch.bfloat16)), "up has the shape"), (dict(down=torch.zeros(4, 8, 16, dtype=torch.bfloat16)), "down has the shape"),
    (dict(router=torch.zeros(16, 4, dtype=torch.bfloat16).t()), "router: the elements"), (dict(gate=torch.zeros(4, 16, 8, dtype=torch.bfloat16).mT), "gate: the elements"),
    (dict(down=torch.zeros(4, 8, 16, dtype=torch.bfloat16).mT), "down: the elements"),
    (dict(gate=torch.zeros(1, 8, 16, dtype=torch.bfloat16).expand(4, 8, 16)), "gate is expanded"),
    (dict(up=torch.zeros(4, 1, 16, dtype=torch.bfloat16).expand(4, 8, 16)), "up is expanded"),
    (dict(router=torch.zeros(1, 16, dtype=torch.bfloat16).expand(4, 16)), "router is expanded"),
    ({}, "on cpu"),
])
def test_experts_of_other_tensors_are_refused(bad, word):
    with pytest.raises(ValueError, match=word):
        experts(**bad)


@pytest.mark.parametrize("bad,word", [
    (torch.zeros(4), "on cpu"), (torch.zeros(4, dtype=torch.bfloat16), "float32"), (torch.zeros(4, dtype=torch.float64), "float32"),
    (torch.zeros(3), "4 query heads"), (torch.zeros(8)[::2], "next to each other"), (torch.zeros(1).expand(4), "next to each other"),
    (L.distance_slopes(4), "on cpu"),
])
@pytest.mark.parametrize("four", [False, True])
def test_slopes_of_other_tensors_are_refused(four, bad, word):
    """distance_slopes() gives a tensor of the host unless it is told a device."""
    c = dict(k=0x10000000, v=0x10000000, dtype=L.BF16, num_pages=8, page_size=16, heads=2, head_dim=64)
    with pytest.raises(ValueError, match=word):
        L.PagedAttention((L.KvCache4 if four else L.KvCache)(**c), 0x10000000, 4, 4, 4, slopes=bad)


def layer():
    """A DecodeAttention's sizes alone: 4 + 2 * 2 heads of 16."""
    it = object.__new__(decode.DecodeAttention)
    it.heads, it.kv_heads, it.head_dim = 4, 2, 16
    it.status = torch.zeros(1)
    return it


@pytest.mark.parametrize("bad,word", [
    (dict(qkv=torch.zeros(5, 128)), "qkv is"), (dict(qkv=torch.zeros(5, 130, dtype=torch.bfloat16)[:, :128]), "qkv is"),
    (dict(qkv=torch.zeros(4, 128, dtype=torch.bfloat16)), "qkv is"), (dict(qkv=torch.zeros(5, 96, dtype=torch.bfloat16)), "qkv is"),
    (dict(k_out=torch.zeros(5, 32, dtype=torch.bfloat16)), "k_out is"), (dict(v_out=torch.zeros(5, 32, dtype=torch.bfloat16)), "v_out is"),
    (dict(k_out=torch.zeros(5, 128)), "k_out is"), (dict(v_out=torch.zeros(4, 128, dtype=torch.bfloat16)), "v_out is"),
    (dict(k_out=torch.zeros(5, 128, dtype=torch.bfloat16)[:, :16]), "k_out is"),
    (dict(pos=torch.zeros(5, dtype=torch.int64)), "pos is"), (dict(seq=torch.zeros(5, dtype=torch.int64)), "seq is"), (dict(pos=torch.zeros(4, dtype=torch.int32)), "pos is"),
])
def test_prompts_of_other_tensors_are_refused(bad, word):
    """Keys and values as held are strided as qkv: rows of their own would be written past their end."""
    a = dict(qkv=torch.zeros(5, 128, dtype=torch.bfloat16), pos=torch.zeros(5, dtype=torch.int32), seq=torch.zeros(5, dtype=torch.int32))
    a.update(bad)
    with pytest.raises(ValueError, match=word):
        layer().prompt(a["qkv"], a["pos"], a["seq"], 5, k_out=a.get("k_out"), v_out=a.get("v_out"))


def test_prompts_of_addresses_and_of_sequences_in_order_reach_the_append():
    """What has no type is the caller's: addresses, and no seq where token t belongs to sequence t."""
    it, got = layer(), []
    it.append = type("Append", (), {"append": lambda self, *a, **kw: got.append((a, kw))})()
    qkv = torch.zeros(1, 130, dtype=torch.bfloat16)[:, :128]  # one row, whose stride says nothing
    it.prompt(qkv, 0x10000000, None, 1, k_out=0x20000000, v_out=0x30000000)
    (a, kw), = got
    assert a[2:] == (0x10000000, 1) and kw["seq"] is None and kw["k_out"] == 0x20000000 and kw["q"] is qkv
