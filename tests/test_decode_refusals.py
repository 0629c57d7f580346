"""Calls of the decoding operators whose arguments are each in range and do not fit each other: refused on the host."""
import pytest

import l2domain_b200 as L

PTR = 0x10000000  # never dereferenced


def append(tokens, q_out, **desc):
    cache = L.KvCache(k=PTR, v=PTR, dtype=L.BF16, num_pages=8, page_size=16, heads=2, head_dim=64)
    d = dict(heads_q=4, cos=PTR, sin=PTR, max_pos=64, rot_dim=64)
    L.KvAppend(cache, PTR, 4, 4, **{**d, **desc}).append(k=PTR, v=PTR, pos=PTR, tokens=tokens, q=PTR, q_out=q_out)


@pytest.mark.parametrize("desc", [dict(q_token=512), dict(q_out_token=512), dict(q_token=512, q_out_token=1024)])
def test_append_in_place_wants_one_stride(desc):
    """Rows of q would be overwritten by other tokens' before they are read."""
    with pytest.raises(L.L2DError, match="q_out is q") as e:
        append(4, PTR, **desc)
    assert e.value.status == -1


@pytest.mark.parametrize("tokens,q_out,desc", [(4, PTR, dict(q_token=512, q_out_token=512)), (4, PTR, dict(q_token=256)),
                                               (1, PTR, dict(q_token=512)), (4, PTR + (1 << 20), dict(q_token=512))])
def test_append_of_other_strides_is_no_refusal(tokens, q_out, desc):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(L.L2DError) as e:
        append(tokens, q_out, **desc)
    assert e.value.status == -3  # no device: every check before has passed


@pytest.mark.parametrize("scale", [3e38, -2.5e38])
def test_attention_scale_must_leave_room_for_its_logarithm(scale):
    """The kernel takes powers of two: a scale whose product with log2(e) is infinite would make 0 * inf of a score of 0."""
    cache = L.KvCache(k=PTR, v=PTR, dtype=L.BF16, num_pages=8, page_size=16, heads=2, head_dim=64)
    with pytest.raises(L.L2DError, match="too large") as e:
        L.PagedAttention(cache, PTR, 4, 4, heads_q=4, scale=scale)
    assert e.value.status == -1
