"""Making a plan of the paged attention beside other work on the GPU."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import l2domain_b200 as L  # noqa: E402
from test_decode_ops_gpu import Pages, attn_check, gpu  # noqa: E402,F401


def test_making_a_plan_waits_for_no_other_stream():
    P = Pages(L.BF16, 2, 20, 16, 2, 64, seed=1)
    attn_check(P, [300, 17], 8, L.BF16)  # kernels are loaded
    busy = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(4_000_000_000)
    plan = L.PagedAttention(P.cache(), P.table, P.seqs, P.width, 8, q_token=8 * 64, out_token=8 * 64)
    assert not busy.query()  # two seconds of it are left
    busy.synchronize()
    attn_check(P, [300, 17], 8, L.BF16, plan=plan)
