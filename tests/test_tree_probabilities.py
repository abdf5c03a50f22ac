"""Which probabilities of a plan with trees are rounded: its items' flags, read as
the kernel reads them, and a model of what rounding them would lose."""
import random

import pytest
import torch

from santa_amd.paged import PagedKVCache, PagedPlan
from santa_amd.runtime import ExactDecodeBackend, LlamaShape, RandomLlama
from test_draft_trees import carry_out, formula, random_tree, seen_tokens
from test_draft_trees_gpu import _reference
from test_paged import _shared_pools

BRANCH = [-1, 0, 0, 1, 1, 2]


def branching(t):
    return [-1] + [max(0, i - 2) for i in range(1, t)]


def chain(t):
    return list(range(-1, t - 1))


def tight(out, ref, dtype, longest, top):
    """The largest share of its bound that a value's error takes, of probabilities in
    two parts; ref: values, mean of |v| and bound of the scores' rounding, top: the largest |v|."""
    want, mean, off = ref
    eps = torch.finfo(dtype).eps / 2
    bound = eps * want.abs() + (4 * eps * eps + off) * (1 + eps) * mean
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 + 2 * longest * 2.0 ** -32 * top
    return ((out.double() - want).abs() / bound.clamp_min(1e-30)).max().item()


def _plan(lens, new, trees, prefixes=(), H=32, KVH=8, **kw):
    return PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new, prefixes=prefixes, parents=trees, device="cpu", **kw)


def in_two_parts(plan):
    """For each sequence the set of its items' flags, own ones and those of prefixes:
    whether probabilities are in two parts."""
    info, data = plan._info, plan._data
    of = [b for b, t in enumerate(plan.new_tokens) for _ in range(t)]
    out = [set() for _ in plan.new_tokens]
    GH = plan.heads // plan.kv_heads
    for w in range(info.groups):
        while w >= 0:
            flags, _, _, _, tok0, rows, _, _, w = data[16 * w:16 * w + 9].tolist()
            two = {0: True, 1: False, 2: bool(flags & 8)}[info.rounded]
            for i in range(rows // GH):
                out[of[int(data[info.list_at + tok0 + i]) if flags & 1 else tok0 + i]].add(two)
    return out


def test_a_tree_does_not_follow_its_neighbours():
    """A small tree is held in two parts alone, beside larger trees and beside a
    prefill, whose own probabilities are rounded."""
    assert in_two_parts(_plan([500], [6], [BRANCH])) == [{True}]
    assert in_two_parts(_plan([500, 900], [6, 25], [BRANCH, branching(25)])) == [{True}, {True}]
    assert in_two_parts(_plan([500, 900], [6, 300], [BRANCH, None])) == [{True}, {False}]
    assert in_two_parts(_plan([500, 900, 70], [64, 300, 1], [branching(64), None, [-1]], H=64)) == [{True}, {False}, {False}]
    # a sequence without a tree, and few rows, does not follow the trees either
    assert in_two_parts(_plan([500, 900], [5, 60], [None, branching(60)])) == [{True}, {True}]
    assert in_two_parts(_plan([500, 900], [1, 60], [None, branching(60)], H=20, KVH=1)) == [{True}, {True}]


def test_prefixes():
    """The rows that trees have in a common prefix are held as their own tokens are,
    beside those of sequences without one."""
    lens, new = [400, 390, 380, 395], [7, 9, 12, 2]
    for fixed in (False, True):
        plan = _plan(lens, new, [branching(7), None, branching(12), None], [([0, 1, 2, 3], 320)], fixed=fixed)
        assert in_two_parts(plan) == [{True}, {False}, {True}, {False}]
        plan = _plan(lens, new, [chain(7), None, [-2] * 12, None], [([0, 1, 2, 3], 320)], fixed=fixed)
        assert in_two_parts(plan) == [{True}, {False}, {True}, {False}]
        plan = _plan(lens, new, [chain(7), chain(9), branching(12), chain(2)], [([0, 1, 2, 3], 320)], fixed=fixed)
        assert in_two_parts(plan) == [{True}] * 4


def test_chains_are_sequences():
    """Trees that are chains are held as without trees."""
    lens, new = [1000, 200, 64], [5, 40, 64]
    plan, plain = _plan(lens, new, [chain(t) for t in new]), PagedPlan(lens, heads=32, kv_heads=8, new_tokens=new, device="cpu")
    assert in_two_parts(plan) == in_two_parts(plain) == [{False}] * 3
    assert in_two_parts(_plan(lens, new, [chain(5), branching(40), branching(64)])) == [{True}] * 3


@pytest.mark.parametrize("prefixes", [[], [([1, 0, 2], 64)]])
def test_updates_keep_the_launch(prefixes):
    """Trees of a fixed plan become chains and others again: the same kernels, with
    items that say how."""
    new, r = [9, 20, 40], random.Random(1)
    plan = _plan([300] * 3, new, [chain(t) for t in new], prefixes, fixed=True)
    first = plan._info

    def launch(info):
        return [getattr(info, n) for n in ("groups", "items", "merge_tokens", "records", "rounded", "tree_ints", "ints",
                                           "pos_at", "tree_at")]

    for lens, trees in (([200, 290, 310], [branching(t) for t in new]), ([104, 150, 299], [chain(9), branching(20), [-2] * 40]),
                        ([104, 150, 110], [random_tree(r, t, 0.2) for t in new]), ([300] * 3, [chain(t) for t in new])):
        plan.update(lens, trees)
        assert launch(plan._info) == launch(first) and plan._info.rounded == 2
        want = [{True} if prefixes or t != chain(len(t)) else {False} for t in trees]
        assert in_two_parts(plan) == want


CASES = [
    ([400, 390, 380, 100], [30, 5, 70, 2], (1,), [([2, 0, 1], 256)], 4, 1, 32),
    ([300, 200, 310, 250, 99], [9, 1, 30, 4, 8], (1, 4), [([3, 0], 200), ([1, 4, 2], 80)], 28, 4, 8),
    ([900, 850, 870, 30], [64, 300, 40, 1], (1, 3), [([0, 1, 2], 512)], 8, 1, 16),
    ([2000 + i for i in range(8)], [40, 1] * 4, (1, 3, 5, 7), [(list(range(8)), 1920)], 4, 2, 16),
]


@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_plans_carried_out(case, fixed):
    """Prefixes whose rows are in two lists, carried out in Python; a row's parts are held alike."""
    lens, new, chains, prefixes, H, KVH, page = CASES[case]
    r = random.Random(case)
    trees = [None if b in chains else random_tree(r, t, 0.1) for b, t in enumerate(new)]
    k, v, table = _shared_pools(lens, prefixes, page, KVH, 16, case)
    q = torch.randn(sum(new), H, 16, generator=torch.Generator().manual_seed(case), dtype=torch.float64)
    plan = _plan(lens, new, trees, prefixes, H, KVH, fixed=fixed)
    assert plan._info.rounded == 2
    want = formula(q, k, v, table, lens, new, trees)
    # float64 sums of up to 2000 terms
    assert torch.allclose(carry_out(q, k, v, table, plan), want, rtol=1e-10, atol=1e-12)
    assert all(len(s) <= 1 for s in in_two_parts(plan))


def test_plans_without_trees_are_as_before():
    for new in ([1, 1], [8, 1], [1, 9], [90, 1, 0, 2], [300]):
        plan = PagedPlan([400] * len(new), heads=8, kv_heads=2, new_tokens=new, device="cpu")
        assert plan._info.rounded == int(max(new) > 8) and not any(f & 8 for f in plan._data[:16 * plan._info.items:16].tolist())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lost", ["nothing", "second", "second product"])
def test_the_bound_holds_two_parts(dtype, lost):
    """The bound of the GPU tests, on a model of the two parts: it holds them, and
    neither probabilities that are rounded once nor a second part that is in the
    mass but not among the products."""
    lens, new = [300, 90], [16, 9]
    r = random.Random(0)
    trees = [random_tree(r, t, 0.1) for t in new]
    k, v, table = _shared_pools(lens, [], 16, 2, 64, 1, dtype=dtype)
    q = torch.randn(25, 8, 64, generator=torch.Generator().manual_seed(2)).mul(1.5).to(dtype)
    want, mean, off = _reference(q, k, v, table, lens, new, trees)
    out, t0 = torch.zeros_like(want), 0
    for b, (n, t) in enumerate(zip(lens, new)):
        for i in range(t):
            at = torch.tensor(seen_tokens(n, t, trees[b], i), dtype=torch.int64)
            if not len(at):
                continue
            kh, vh = (x[table[b, at // 16].long(), at % 16].double().repeat_interleave(4, 1) for x in (k, v))
            s = (kh * q[t0 + i].double()).sum(-1) / 8.0
            e = torch.exp(s - s.amax(0)) * (1.0 if dtype == torch.bfloat16 else 128.0)
            p = e.to(dtype).double()
            low = (e - p).to(dtype).double()
            used = p if lost != "nothing" else p + low
            mass = p if lost == "second" else p + low
            out[t0 + i] = (used[..., None] * vh).sum(0) / mass.sum(0)[:, None]
        t0 += t
    share = tight(out.to(dtype), (want, mean, off), dtype, max(lens), v.nan_to_num(0.0).abs().max().item())
    assert share <= 1 if lost == "nothing" else share > 1


def test_extend_takes_the_choice():
    """The model hands `rounded` on; a backend has its own way."""
    shape = LlamaShape(hidden=64, intermediate=64, heads=4, kv_heads=2, layers=1, vocab=50)
    model = RandomLlama(shape, seed=1, device="cpu", dtype=torch.float32)
    cache = PagedKVCache(1, 20, 8, kv_heads=2, head_dim=16, max_seqs=2, max_len=80, dtype=torch.float32, device="cpu")
    s, = cache.add([0])
    tokens = torch.arange(20)
    want = model.extend(tokens[None], cache, [s], rounded=False)
    t, = cache.add([0])
    assert torch.equal(model.extend(tokens[None], cache, [t]), want)
    with pytest.raises(ValueError, match="own way"):
        model.extend(tokens[:1, None], cache, [s], backend=ExactDecodeBackend(), rounded=True)
    assert cache.lengths([s]) == [20]
