"""Plans of shared paged caches on streams other than the one they were made on,
and in captured graphs.

Every case prints its name before touching the GPU.
"""
import pytest
import torch

from santa_amd.paged import PagedPlan, paged_attention, rope_append
from test_shared_pages_gpu import _case, _check, _reference

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
        torch.cuda._sleep(1_000_000_000)  # about 0.4 s
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


def _capture(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


@pytest.mark.parametrize("new, H, KVH, D, dtype", [([1] * 4, 8, 2, 128, BF), ([1] * 4, 40, 1, 64, torch.float16),
                                                   ([3, 1, 20, 2], 4, 1, 128, BF)])
def test_replays_follow_the_plan(new, H, KVH, D, dtype):
    """Replays after updates against the formula on the lengths then in force:
    the shortest that the prefix allows, the longest that the table holds, and
    none beyond it."""
    print(f"\n[case] replays against the formula, new={new} H={H} D={D} {dtype}", flush=True)
    page, longest = 16, [900, 640, 333, 800]
    shared = [([0, 3], 192)]
    q, k, v, table, _ = _case(longest, new, shared, H, KVH, D, page, dtype, 3)
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.5)
    table = table.clamp(0, k.shape[0] - 1)
    room = table.shape[1] * page
    plan = PagedPlan([200 + t for t in new], heads=H, kv_heads=KVH, new_tokens=new, prefixes=shared, fixed=True)
    cs = torch.randn(2, sum(new), D, device="cuda").to(dtype)
    qkv = torch.randn(sum(new), H + 2 * KVH, D, device="cuda").to(dtype)

    def step():
        turned = rope_append(qkv, cs[0], cs[1], k, v, table, plan)
        return turned, paged_attention(turned, k, v, table, plan)

    graph, (turned, out) = _capture(step)
    with pytest.raises(RuntimeError, match=f"{room + 1} > {room}"):
        plan.update([200 + t for t in new[:3]] + [room + 1])
    for lens in ([192 + new[0], 0, 1, 192 + new[3]], longest, [room - 7, 64, 128 + new[2], 700], [500, 65, 20, 192 + 64]):
        plan.update(lens)
        qkv.normal_()
        out.zero_()
        graph.replay()
        # rows of the formula in the order of the plan; appended tokens are in the pools by then
        _check(out, _reference(turned, k, v, table, lens, new), dtype)
        assert torch.equal(out, paged_attention(turned, k, v, table, plan))


def test_plans_that_replays_do_not_follow():
    """A plan that is not fixed, and expressions, which hold its lengths: no update
    behind a capture."""
    print("\n[case] captured plans without updates", flush=True)
    for dtype, fixed in ((BF, False), (torch.float32, True)):
        q, k, v, table, plan = _case([100, 64], [1, 1], [], 4, 2, 64, 16, dtype, fixed=fixed)
        graph, out = _capture(lambda: paged_attention(q, k, v, table, plan))
        with pytest.raises(RuntimeError, match="a captured call holds"):
            plan.update([50, 64])
        for _ in range(3):
            q.normal_()
            graph.replay()
            assert torch.equal(out, paged_attention(q, k, v, table, plan))
