"""Trees of drafted tokens over shared paged caches, on the CPU: plans carried out
in Python as the kernels carry them out, the torch expressions and their
gradients, and refusals.
"""
import ctypes
import math
import random

import pytest
import torch

from santa_amd import paged
from santa_amd.paged import PagedPlan, paged_attention, rope_append
from test_paged import _shared_pools


def random_tree(r, t, unused=0.0):
    """Parents of t drafted tokens, some not in use (and followed by none)."""
    parents = []
    for i in range(t):
        before = [-1] + [j for j in range(i) if parents[j] != -2]
        parents.append(-2 if r.random() < unused else r.choice(before[-4:] + [r.choice(before)]))
    return parents


def path(parents, i):
    """Token i and those that it follows."""
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


def seen_tokens(n, t, parents, i):
    """The places that new token i of a sequence attends to, [] where it is not in use."""
    if parents is None:
        return list(range(n - t + i + 1))
    if n < t or parents[i] == -2:
        return []
    return list(range(n - t)) + [n - t + j for j in path(parents, i)]


def formula(q, k, v, table, lens, new, trees):
    """Token by token in float64."""
    N, H, D = q.shape
    page, KVH = k.shape[1:3]
    out, t0 = torch.zeros(N, H, D, dtype=torch.float64), 0
    for b, (n, t) in enumerate(zip(lens, new)):
        for i in range(t):
            at = torch.tensor(seen_tokens(n, t, trees[b], i), dtype=torch.int64)
            if len(at):
                ks, vs = (x[table[b, at // page].long(), at % page].double() for x in (k, v))
                for h in range(H):
                    p = torch.softmax(ks[:, h // (H // KVH)] @ q[t0 + i, h].double() / math.sqrt(D), 0)
                    out[t0 + i, h] = p @ vs[:, h // (H // KVH)]
        t0 += t
    return out


def carry_out(q, k, v, table, plan):
    """The plan as the kernels carry it out: every item's parts with its rows'
    limits or bits, then the join."""
    info, data = plan._info, plan._data
    H, KVH, page, D = plan.heads, plan.kv_heads, k.shape[1], q.shape[2]
    GH, N = H // KVH, plan.tokens
    out = torch.full((N, H, D), math.nan, dtype=torch.float64)
    part, written = {}, set()
    for w in range(info.groups):
        while w >= 0:
            flags, row, begin, end, tok0, rows, pos0, base, w, tree0 = data[16 * w:16 * w + 10].tolist()
            if rows == 0:
                continue
            at = torch.arange(begin, end)
            kk, vv = (x[table[row, at // page].long(), at % page] for x in (k, v))
            for r in range(rows):
                tok = int(data[info.list_at + tok0 + r // GH]) if flags & 1 else tok0 + r // GH
                seen, blind = at <= pos0 + r // GH, pos0 + r // GH < 0
                if flags & 4:
                    record = data[info.tree_at + tok * info.tree_ints:][:info.tree_ints].tolist()
                    blind = record[1] < 0
                    seen = torch.ones(len(at), dtype=torch.bool)
                    for x in range(begin, end):
                        if x // 64 >= tree0 // 64:
                            bit = x - tree0 // 64 * 64
                            seen[x - begin] = record[2 + bit // 32] >> (bit % 32) & 1
                for kv in range(KVH):
                    h = kv * GH + r % GH
                    s = (kk[:, kv] @ q[tok, h] / math.sqrt(D))[seen]
                    m = s.max() if len(s) else torch.tensor(-3.4e38, dtype=torch.float64)
                    e = torch.exp(s - m)
                    res = (m, e.sum(), e @ vv[seen, kv])
                    if flags & 2:
                        assert (tok, h) not in written
                        written.add((tok, h))
                        out[tok, h] = 0.0 if blind else res[2] / res[1]
                    else:
                        rec = base + kv * rows + r
                        assert rec not in part and rec < info.records
                        part[rec] = res
    for j in range(info.merge_tokens):
        tok = int(data[info.merge_at + j])
        a, b = data[info.parts_at + 8 * tok:info.parts_at + 8 * tok + 8].view(2, 4).tolist() if tok >= 0 else (0, [0] * 4)
        if b[3] == 0:
            continue
        for h in range(H):
            ps = [part.pop(p[0] + (s * KVH + h // GH) * p[1] + p[2] + h % GH) for p in (a, b) for s in range(p[3])]
            top = max(p[0] for p in ps)
            w = [torch.exp(p[0] - top) for p in ps]
            assert (tok, h) not in written
            written.add((tok, h))
            blind = int(data[info.pos_at + 2 * tok]) < 0
            out[tok, h] = 0.0 if blind else sum(x * p[2] for x, p in zip(w, ps)) / sum(x * p[1] for x, p in zip(w, ps))
    assert not part and len(written) == N * H
    return out


PLANS = [
    # lens, new tokens, sequences without a tree, share not in use, prefixes, H, KVH, page
    ([1], [1], (), 0.0, [], 4, 2, 8),
    ([9, 64, 65, 128], [8, 64, 1, 3], (), 0.0, [], 2, 2, 8),
    ([130, 131, 200], [5, 2, 9], (1,), 0.2, [([0, 1, 2], 120)], 4, 1, 16),
    ([130, 131, 200, 90], [3, 70, 60, 1], (), 0.3, [([2, 0], 120), ([3, 1], 60)], 6, 2, 8),
    ([300, 20, 2, 0], [5, 20, 7, 3], (), 0.2, [], 4, 2, 8),
    ([300, 20, 2, 5], [250, 20, 7, 0], (2,), 0.1, [], 7, 1, 32),
    ([2000], [129], (), 0.5, [], 8, 2, 64),
    ([], [], (), 0.0, [], 4, 2, 8),
    ([700, 900], [40, 60], (), 0.1, [], 8, 1, 16), ([900, 20, 66], [40, 60, 33], (1,), 0.0, [], 8, 1, 16),
]


def _case(case, fixed=False, trees=None):
    lens, new, chains, unused, prefixes, H, KVH, page = PLANS[case]
    r = random.Random(case)
    trees = [None if b in chains else random_tree(r, t, unused) for b, t in enumerate(new)] if trees is None else trees
    k, v, table = _shared_pools(lens, prefixes, page, KVH, 16, case)
    q = torch.randn(sum(new), H, 16, generator=torch.Generator().manual_seed(case), dtype=torch.float64)
    plan = PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new, prefixes=prefixes, device="cpu", fixed=fixed,
                     parents=trees)
    return q, k, v, table, plan, trees


@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("case", range(len(PLANS)))
def test_plan(case, fixed):
    """Carried out, a plan gives every token the attention of what it follows; the
    expressions do the same, and positions are those behind the token followed."""
    q, k, v, table, plan, trees = _case(case, fixed)
    want = formula(q, k, v, table, plan.seq_lens, plan.new_tokens, trees)
    assert (carry_out(q, k, v, table, plan) - want).abs().sum() < 1e-9 * max(1, want.numel())
    assert (paged_attention(q, k, v, table, plan) - want).abs().sum() < 1e-9 * max(1, want.numel())
    pos = [len(seen_tokens(n, t, p, i)) - 1 if p is not None else n - t + i
           for n, t, p in zip(plan.seq_lens, plan.new_tokens, trees) for i in range(t)]
    assert plan.positions.tolist() == pos


def test_chains_are_sequences():
    """Trees that are chains give a plan's own bits."""
    lens, new = [130, 77], [5, 40]
    k, v, table = _shared_pools(lens, [], 8, 2, 16, 3)
    q = torch.randn(45, 4, 16, dtype=torch.float64)
    args = dict(heads=4, kv_heads=2, new_tokens=new, device="cpu")
    tree = PagedPlan(lens, parents=[list(range(-1, t - 1)) for t in new], **args)
    plain = PagedPlan(lens, **args)
    assert torch.equal(tree.positions, plain.positions)
    assert torch.allclose(paged_attention(q, k, v, table, tree), paged_attention(q, k, v, table, plain), atol=1e-12)


@pytest.mark.parametrize("fixed", [False, True])
def test_update(fixed):
    """Other lengths, with the trees as they were or others of as many tokens."""
    lens, new, r = [130, 70, 64], [9, 3, 30], random.Random(0)
    trees = [random_tree(r, 9), None, random_tree(r, 30)]
    plan = PagedPlan(lens, heads=4, kv_heads=2, new_tokens=new, device="cpu", fixed=fixed, parents=trees)
    size = len(plan._data)
    for lens, other in (([200, 71, 31], None), ([127, 3, 64], [random_tree(r, 9, 0.3), None, random_tree(r, 30, 0.3)]),
                        ([0, 0, 29], None)):
        plan.update(lens, other)
        trees = other or trees
        k, v, table = _shared_pools(lens, [], 8, 2, 16, 1)
        q = torch.randn(42, 4, 16, dtype=torch.float64)
        want = formula(q, k, v, table, lens, new, trees)
        assert (carry_out(q, k, v, table, plan) - want).abs().max() < 1e-9
        assert not fixed or len(plan._data) == size
    before = (plan._data.clone(), plan.seq_lens, plan.parents)
    for bad in ([trees[0], trees[0][:3], trees[2]], [trees[0], None], [trees[0][:8], None, trees[2]], [None, None, trees[2]]):
        with pytest.raises(ValueError):
            plan.update(lens, bad)
    with pytest.raises(RuntimeError, match="is an earlier one"):
        plan.update(lens, [[0] * 9, None, trees[2]])
    assert torch.equal(plan._data, before[0]) and (plan.seq_lens, plan.parents) == before[1:]
    with pytest.raises(ValueError, match="without trees"):
        PagedPlan([5], heads=1, kv_heads=1, device="cpu").update([5], [[-1]])


def test_refusals():
    make = lambda parents, t=3, n=20: PagedPlan([n], heads=2, kv_heads=1, new_tokens=t, device="cpu",  # noqa: E731
                                                parents=parents)
    for parents, text in (([[-1, 1, 0]], "is an earlier one"), ([[-1, 0, -3]], "is an earlier one"),
                          ([[-1, -2, 1]], "which is not in use"), ([[0, 0, 0]], "is an earlier one")):
        with pytest.raises(RuntimeError, match=text):
            make(parents)
    for parents in ([[-1, 0]], [[-1, 0, 0], None], [[-1, 0, 0.5]], [5], [None, None]):
        with pytest.raises((ValueError, TypeError)):
            make(parents)
    assert make([list(range(-1, 8191))], 8192, 9000).tokens == 8192
    with pytest.raises(RuntimeError, match="up to 8192"):
        make([list(range(-1, 8192))], 8193, 9000)
    with pytest.raises(RuntimeError, match="beside trees"):
        PagedPlan([2000, 1 << 21], heads=1, kv_heads=1, new_tokens=[1024, 1 << 21], device="cpu",
                  parents=[[-1] * 1024, None])
    lib, info = paged._lib(), paged._PlanInfo()
    one = (ctypes.c_int * 1)(1)
    assert lib.santa_paged_tree_plan(one, one, None, 1, None, None, 0, 1, 1, 0, None, None, ctypes.byref(info), None, 0) == 1
    assert b"santa_paged_tree_plan" in lib.santa_last_error()


def test_unused_tokens_are_not_written():
    k, v, table = _shared_pools([20, 3], [], 8, 1, 16, 2)
    trees = [[-1, -2, 0, -2], [-1, 0, 0, 1]]
    plan = PagedPlan([20, 3], heads=2, kv_heads=1, new_tokens=4, device="cpu", parents=trees)
    qkv, cs = torch.randn(8, 4, 16, dtype=torch.float64), torch.ones(8, 16, dtype=torch.float64)
    k2, v2 = k.clone(), v.clone()
    rope_append(qkv, cs, 0 * cs, k2, v2, table, plan)
    for i in (16, 18):
        at = (table[0, i // 8].long(), i % 8)
        assert torch.equal(k2[at], qkv[i - 16, 2:3]) and torch.equal(v2[at], qkv[i - 16, 3:])
        k2[at], v2[at] = k[at], v[at]
    assert torch.equal(k2.nan_to_num(7), k.nan_to_num(7)) and torch.equal(v2.nan_to_num(7), v.nan_to_num(7))


def test_masked_values_stay_out():
    """Infinities and NaN in drafted tokens reach those that follow them only."""
    lens, new = [70, 66], [6, 4]
    trees = [[-1, 0, 0, 1, 1, 2], [-1, -1, 0, -2]]
    k, v, table = _shared_pools(lens, [], 8, 1, 16, 4)
    q = torch.randn(10, 2, 16, dtype=torch.float64)
    plan = PagedPlan(lens, heads=2, kv_heads=1, new_tokens=new, device="cpu", parents=trees)
    for t, bad in ((1, math.nan), (2, math.inf), (4, -math.inf)):
        n = 64 + t
        v[table[0, n // 8].long(), n % 8] = bad
        if t != 2:
            k[table[0, n // 8].long(), n % 8] = math.nan
    v[table[1, 65 // 8].long(), 65 % 8] = math.nan  # not in use
    k[table[1, 65 // 8].long(), 65 % 8] = math.inf
    out = paged_attention(q, k, v, table, plan)
    assert torch.isfinite(out[0]).all() and out[[1, 3, 4]].isnan().all() and (out[[2, 5]] == math.inf).all()
    assert torch.isfinite(out[6:]).all() and (out[9] == 0).all()


def test_expressions_differentiate():
    """Gradients of q, k and v against differences; a token not in use has none."""
    lens, new, trees = [13, 9], [4, 3], [[-1, 0, 0, -2], [-1, 0, 1]]
    k, v, table = (t.nan_to_num(0.0) if t.is_floating_point() else t for t in _shared_pools(lens, [], 8, 1, 4, 5))
    q = torch.randn(7, 2, 4, dtype=torch.float64)
    plan = PagedPlan(lens, heads=2, kv_heads=1, new_tokens=new, device="cpu", parents=trees)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    assert torch.autograd.gradcheck(lambda q, k, v: paged_attention(q, k, v, table, plan), leaves)
    g, = torch.autograd.grad(paged_attention(*leaves, table, plan).sum(), leaves[:1])
    assert (g[3] == 0).all()
