"""Plans of shared paged caches on streams other than the one they were made on,
and in captured graphs.

Every case prints its name before touching the GPU.
"""
import gc

import pytest
import torch

from santa_amd.paged import paged_attention, rope_append
from test_shared_pages_gpu import _case

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("end", ["dropped", "updated", "updated on the stream"])
@pytest.mark.parametrize("call", ["attention", "append", "update"])
def test_a_plan_outlives_its_calls(call, end):
    """A plan that is dropped or given other lengths while a call on another
    stream is still to run keeps its memory until that call has ended."""
    print(f"\n[case] plan used on another stream by {call}, {end}", flush=True)
    lens = [300, 90]
    q, k, v, table, plan = _case(lens, [1, 1], [], 8, 2, 128, 16, BF)
    qkv, cs = torch.randn(2, 12, 128, device="cuda").bfloat16(), torch.ones(2, 128, device="cuda", dtype=BF)
    want = paged_attention(q, k, v, table, plan)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about 0.1 s
        if call == "attention":
            got = paged_attention(q, k, v, table, plan)
        elif call == "append":
            rope_append(qkv, cs, cs, k.clone(), v.clone(), table, plan)
        else:
            plan.update(lens)
        busy = torch.cuda.Event()
        busy.record()
    at, size = plan._data.data_ptr(), plan._data.numel()
    if end == "dropped":
        del plan
        gc.collect()
    elif end == "updated":
        plan.update([30000, 9])  # more work: a plan of another size
    else:
        with torch.cuda.stream(side):
            plan.update([30000, 9])
    others = [torch.full((size,), -1, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert not busy.query() and all(t.data_ptr() != at for t in others)
    torch.cuda.synchronize()
    if call == "attention":
        assert torch.equal(got, want)
