"""Rules on logits on the GPU: against the formula in float64 (tests/test_logits.py)
where it is small, and bit for bit against the expressions on the CPU, whose float32
operations are the kernel's in the same order.  Every case prints its name before
touching the GPU."""
import math
import random

import pytest
import torch

from santa_amd.logits import adjust_logits
from santa_amd.paged import PagedPlan
from test_draft_trees import random_tree
from test_logits import ALL, CASES, check, formula, make, random_rules

pytestmark = pytest.mark.gpu


def cuda(x):
    if isinstance(x, tuple):
        return tuple(map(cuda, x))
    return x.cuda() if isinstance(x, torch.Tensor) else x


def on_gpu(plan, **kw):
    return PagedPlan(plan.seq_lens, heads=4, kv_heads=2, new_tokens=plan.new_tokens, rows=plan.rows,
                     parents=plan.parents, **kw)


def same(logits, tokens, plan, kw, **more):
    """The GPU's values are the CPU's; greedy, the tokens of their maxima."""
    want = adjust_logits(logits, tokens, plan, **kw)
    dev, args = on_gpu(plan, **more), {k: cuda(v) for k, v in kw.items()}
    out = adjust_logits(logits.cuda(), cuda(tokens), dev, **args)
    assert out.dtype == torch.float32 and torch.equal(out.cpu(), want)
    token = adjust_logits(logits.cuda(), cuda(tokens), dev, greedy=True, **args)
    assert token.dtype == torch.int64 and torch.equal(token.cpu(), want.argmax(-1))
    return out


@pytest.mark.parametrize("kinds", [ALL, ("repetition",), ("frequency", "prompts"), ("bias",), ("allowed",), ()])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_rules(case, kinds):
    print(f"\n[case] rules {case} {kinds}", flush=True)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits, tokens, plan, kw = make(case, kinds, dtype)
        check(same(logits, tokens, plan, kw).cpu(), formula(logits, tokens, plan, **kw))
        same(logits, tokens.long(), plan, kw, fixed=True)
        same(logits, None, plan, kw)


def large(lens, new, V, K, seed, chains=(), dtype=torch.float32, trees=True):
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    parents = [None if b in chains else random_tree(r, t, 0.1) for b, t in enumerate(new)] if trees else None
    plan = PagedPlan(lens, heads=4, kv_heads=2, new_tokens=new, parents=parents, device="cpu")
    N, S = sum(new), len(lens)
    logits = (torch.randn(N, V, generator=g) * 3).to(dtype)
    tokens = (V ** torch.rand(S, max(lens), generator=g, dtype=torch.float64)).to(torch.int32) % V
    return logits, tokens, plan, random_rules(g, r, V, S, N, K, ALL)


@pytest.mark.parametrize("lens, new, V, K, chains, dtype, trees", [
    ([3000], [1], 128256, 300, (), torch.float32, False), ([5000, 70, 900], [1, 1, 1], 128256, 2046, (), torch.bfloat16, False),
    ([200 + 31 * i for i in range(12)], [25] * 12, 32001, 20, (3, 7), torch.float32, True),  # rows that are not aligned
    ([700, 800, 900], [64, 100, 1], 50002, 50, (1,), torch.float16, True),
    ([300 + i for i in range(40)], [40] * 40, 4100, 9, (), torch.float32, True),  # many rows to a workgroup
    ([90] * 600, [1] * 600, 2049, 5, (), torch.float32, False), ([1100], [1024], 1000, 5, (), torch.float32, True),
    ([60000], [3], 100, 5, (), torch.float32, True), ([9000], [8192], 40, 5, (), torch.float16, True),
])
def test_sizes(lens, new, V, K, chains, dtype, trees):
    print(f"\n[case] sizes lens={lens[:4]} new={new[:4]} V={V} K={K} {dtype}", flush=True)
    same(*large(lens, new, V, K, V, chains, dtype, trees))


def test_many_rows():
    """More rows than a grid has in one dimension, of one sequence each and without any."""
    print("\n[case] many rows", flush=True)
    x = torch.randn(140001, 9, device="cuda")
    assert torch.equal(adjust_logits(x), x) and torch.equal(adjust_logits(x, greedy=True), x.argmax(-1))
    t = torch.randint(0, 9, (140001, 4), device="cuda", dtype=torch.int32)
    out = adjust_logits(x, t, [3] * 140001, presence=2.0)
    seen = torch.zeros_like(x, dtype=torch.bool).scatter_(1, t[:, :3].long(), True)
    assert torch.equal(out, torch.where(seen, x - 2.0, x))


def test_the_same_row_twice():
    """Entries of a batch that read one row of the table, with other lengths, trees or
    none, one after the other in a workgroup."""
    print("\n[case] the same row twice", flush=True)
    r = random.Random(7)
    lens, new = [130, 70, 66, 200, 66, 500, 66], [30, 6, 2, 9, 30, 1, 5]
    trees = [random_tree(r, 30, 0.1), random_tree(r, 6), random_tree(r, 2), None, random_tree(r, 30), None, random_tree(r, 5)]
    rows = [0, 0, 0, 0, 0, 0, 0]
    g = torch.Generator().manual_seed(0)
    tokens = torch.randint(0, 50, (1, 520), generator=g, dtype=torch.int32)
    for V in (50, 128256):
        logits = torch.randn(sum(new), V, generator=g)
        plan = PagedPlan(lens, heads=4, kv_heads=2, new_tokens=new, rows=rows, parents=trees, device="cpu")
        kw = dict(repetition=1.2, frequency=0.1, prompts=torch.tensor([40], dtype=torch.int32))
        same(logits, tokens, plan, kw)
    big = [[-1] + [0] * 599, [-1] + [0] * 599]  # drafts beyond a workgroup's lanes
    plan = PagedPlan([700, 664], heads=4, kv_heads=2, new_tokens=600, rows=[0, 0], parents=big, device="cpu")
    same(torch.randn(1200, 64, generator=g), torch.randint(0, 64, (1, 700), generator=g, dtype=torch.int32), plan,
         dict(presence=0.5, frequency=0.25))


def test_layouts():
    """Rows that lie apart, columns that do, tables that are views, one row for all."""
    print("\n[case] layouts", flush=True)
    logits, tokens, plan, kw = large([90, 70], [9, 4], 1000, 7, 1)
    want = adjust_logits(logits, tokens, plan, **kw)
    dev, args = on_gpu(plan), {k: cuda(v) for k, v in kw.items()}
    x, t = logits.cuda(), tokens.cuda()
    for y in (torch.cat([x, x], 1)[:, :1000], torch.cat([x[:, :1], x], 1)[:, 1:], x.t().contiguous().t(),
              torch.stack([x, x], -1)[..., 0]):
        for z in (t, t.long(), torch.cat([t, t], 1)[:, :t.shape[1]], t.t().contiguous().t()):
            assert torch.equal(adjust_logits(y, z, dev, **args).cpu(), want)
            assert torch.equal(adjust_logits(y, z, dev, greedy=True, **args).cpu(), want.argmax(-1))
    args["bias"] = tuple(b.t().contiguous().t() for b in args["bias"])
    args["allowed"] = torch.stack([args["allowed"]] * 2, -1)[..., 0]
    args["prompts"] = torch.stack([args["prompts"]] * 2, -1)[..., 0]
    args = {k: torch.stack([v] * 2, -1)[..., 0] if isinstance(v, torch.Tensor) and v.dim() == 1 else v for k, v in args.items()}
    assert torch.equal(adjust_logits(x, t, dev, **args).cpu(), want)
    one = torch.randn(1, 77)  # strides of single rows are never used
    assert torch.equal(adjust_logits(one.cuda().as_strided((1, 77), (3, 1))).cpu(), one)


def test_not_finite():
    print("\n[case] not finite", flush=True)
    x = torch.tensor([[math.nan, 1.0, -math.inf, math.inf], [math.nan, 2.0, 3.0, 3.0], [-math.inf] * 4, [-0.0, 0.0, -1.0, 0.0],
                      [-1.0, math.nan, math.nan, 5.0]]).cuda()
    bits = torch.tensor([[0b0110], [0b1110], [0b1111], [0b1111], [0b1111]], dtype=torch.int32).cuda()
    out = adjust_logits(x, torch.tensor([[0, 1, 2, 3]] * 5).cuda(), [4, 2, 4, 4, 0], repetition=2.0, allowed=bits)
    assert out[0].tolist() == [-math.inf, 0.5, -math.inf, -math.inf] and out[1].tolist() == [-math.inf, 1.0, 3.0, 3.0]
    assert adjust_logits(x, greedy=True).tolist() == [0, 0, 0, 0, 1] == x.argmax(-1).tolist()
    assert adjust_logits(x, allowed=bits, greedy=True).tolist() == [1, 2, 0, 0, 1]
    assert adjust_logits(x, allowed=bits * 0, greedy=True).tolist() == [0] * 5


def test_autograd_and_other_types_take_the_expressions():
    print("\n[case] expressions", flush=True)
    logits, tokens, plan, kw = large([90, 70], [9, 4], 300, 7, 1)
    dev, args = on_gpu(plan), {k: cuda(v) for k, v in kw.items()}
    x = logits.cuda().requires_grad_()
    out = adjust_logits(x, tokens.cuda(), dev, **args)
    # torch's quotient by a number is a product with its inverse there: a rounding more
    check(out.detach().cpu(), formula(logits, tokens, plan, **kw), roundings=6)
    out[torch.isfinite(out)].sum().backward()
    assert x.grad.abs().sum() > 0
    double = adjust_logits(logits.cuda().double(), tokens.cuda(), dev, **args)
    want, _ = formula(logits, tokens, plan, **kw)
    at = torch.isfinite(want)
    assert double.dtype == torch.float64 and (double.cpu() - want)[at].abs().max() < 1e-9


def test_streams_and_replays():
    """On a stream of its own, and captured, values and tokens: replays follow the
    plan's updates, the tokens and the rules that lie in the same memory."""
    print("\n[case] streams and replays", flush=True)
    logits, tokens, plan, kw = large([90, 70, 200], [9, 4, 16], 40000, 7, 1)
    dev, args = on_gpu(plan, fixed=True), {k: cuda(v) for k, v in kw.items()}
    x, t = logits.cuda(), tokens.cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        aside = adjust_logits(x, t, dev, **args)
    side.synchronize()
    assert torch.equal(aside.cpu(), adjust_logits(logits, tokens, plan, **kw))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = adjust_logits(x, t, dev, **args)
        token = adjust_logits(x, t, dev, greedy=True, **args)
    r = random.Random(0)
    for lens, trees in (([90, 70, 200], None), ([200, 4, 64], [random_tree(r, n, 0.2) for n in (9, 4, 16)]), ([8, 0, 199], None)):
        dev.update(lens, trees)
        plan.update(lens, trees)
        x.copy_(torch.randn_like(x))
        t.copy_(t.flip(1))
        graph.replay()
        torch.cuda.synchronize()
        want = adjust_logits(x.cpu(), t.cpu(), plan, **kw)
        assert torch.equal(out.cpu(), want) and torch.equal(token.cpu(), want.argmax(-1))
    with pytest.raises(RuntimeError, match="exceeds"):
        dev.update([201, 4, 64])
