"""A plan's positions, which are its own memory, in captured graphs and on other
streams.  Every case prints its name before touching the GPU."""
import pytest
import torch

from santa_amd.paged import PagedPlan, rope_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("trees", [None, [[-1, 0, 0], None, [-1, -2]]])
def test_captured_positions(trees):
    """Replays follow a fixed plan's updates; another plan is not updated, as its
    memory may not be what the graph reads."""
    print(f"\n[case] captured positions trees={trees is not None}", flush=True)
    kw = dict(heads=4, kv_heads=2, new_tokens=[3, 1, 2], parents=trees)
    plan = PagedPlan([30, 5, 9], fixed=True, **kw)
    rope_tables(plan.positions, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cos, sin = rope_tables(plan.positions, 64)
    for lens in ([30, 5, 9], [100, 2000, 64], [3, 1, 2]):
        plan.update(lens)
        graph.replay()
        torch.cuda.synchronize()
        want = rope_tables(PagedPlan(lens, device="cpu", **kw).positions.cuda(), 64)
        assert torch.equal(cos, want[0]) and torch.equal(sin, want[1])
    loose = PagedPlan([30, 5, 9], **kw)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        rope_tables(loose.positions, 64)
    with pytest.raises(RuntimeError, match="fixed=True"):
        loose.update([100, 2000, 64])
    free = PagedPlan([30, 5, 9], **kw)
    rope_tables(free.positions, 64)
    free.update([100, 2000, 64])
    assert torch.equal(free.positions.cpu(), PagedPlan([100, 2000, 64], device="cpu", **kw).positions)


def test_positions_on_another_stream():
    """Read on another stream, the memory is not given out again before that ends."""
    print("\n[case] positions on another stream", flush=True)
    lens = list(range(1000, 1000 + 64))
    plan = PagedPlan(lens, heads=4, kv_heads=2)
    data, calls = plan._data, []

    class Noted:
        shape = data.shape

        def record_stream(self, stream):
            calls.append(stream)

        def __getitem__(self, at):
            return data[at]

    plan._data = Noted()
    assert torch.equal(plan.positions.cpu(), torch.tensor(lens, dtype=torch.int32) - 1) and not calls
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        at = plan.positions
    side.synchronize()
    assert calls == [side] and torch.equal(at.cpu(), torch.tensor(lens, dtype=torch.int32) - 1)
