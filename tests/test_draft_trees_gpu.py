"""Trees of drafted tokens over shared paged caches on the GPU, against float64.

Tolerance: that of the paged attention (tests/test_shared_pages_gpu.py): the output
is rounded once, the probabilities once more or, with at most 16 rows to a KV head,
twice as finely; float32 scores.

Every case prints its name before touching the GPU.
"""
import math
import random

import pytest
import torch

from santa_amd.paged import PagedPlan, paged_attention
from test_draft_trees import random_tree, seen_tokens
from test_paged import _shared_pools
from test_shared_pages_gpu import _check

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def _reference(q, k, v, table, lens, new, trees):
    """(values, mean of |v|, bound of the scores' rounding) in float64, token by token."""
    N, H, D = q.shape
    page, KVH = k.shape[1:3]
    out, mean, off = (torch.zeros(N, H, D, dtype=torch.float64, device=q.device) for _ in range(3))
    t0 = 0
    for b, (n, t) in enumerate(zip(lens, new)):
        every = torch.arange(n, device=q.device)
        rows = (table[b, every // page].long(), every % page)
        ks, vs = k[rows], v[rows]
        for i in range(t):
            at = torch.tensor(seen_tokens(n, t, trees[b], i), dtype=torch.int64, device=q.device)
            if not len(at):
                continue
            kh, vh = (x[at].double().repeat_interleave(H // KVH, 1) for x in (ks, vs))  # [seen, H, D]
            x = q[t0 + i].double()
            p = torch.softmax((kh * x).sum(-1) / math.sqrt(D), 0)[..., None]
            out[t0 + i], mean[t0 + i] = (p * vh).sum(0), (p * vh.abs()).sum(0)
            size = (kh * x).abs().sum(-1).amax(0) / math.sqrt(D)
            off[t0 + i] = (2 * (D + 2) * 2.0 ** -24 * size + 2.0 ** -20)[:, None]
        t0 += t
    return out, mean, off


def _case(lens, new, trees, prefixes, H, KVH, D, page, dtype, seed=0, **kw):
    k, v, table = (t.cuda() for t in _shared_pools(lens, prefixes, page, KVH, D, seed, dtype=dtype))
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(sum(new), H, D, generator=g).mul(1.5).to("cuda", dtype)
    plan = PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new, prefixes=prefixes, parents=trees, **kw)
    return q, k, v, table, plan


# contexts around the tiles of 64, pages that end inside one, trees of one token to
# more than a tile, tokens not in use, batches with sequences without trees, and
# every row count from one to several blocks of 256
CASES = [
    # lens, new, sequences without a tree, share not in use, prefixes, H, KVH, D, page, dtype
    ([1], [1], (), 0.0, [], 8, 2, 128, 16, BF), ([64], [1], (), 0.0, [], 4, 4, 64, 8, F16),
    ([72, 63 + 9, 65 + 9, 9], [8, 9, 9, 9], (), 0.0, [], 2, 1, 128, 8, BF),
    ([128 + 3, 127 + 3, 5], [3, 3, 5], (), 0.2, [], 4, 1, 64, 16, F16),
    ([700, 20, 0], [16, 16, 16], (), 0.2, [], 4, 2, 128, 32, BF), ([1000], [8], (), 0.0, [], 32, 8, 128, 16, BF),
    ([500, 400], [12, 5], (1,), 0.0, [], 40, 1, 64, 16, F16), ([300, 65], [64, 64], (), 0.1, [], 4, 1, 128, 256, BF),
    ([300, 200], [65, 130], (), 0.1, [], 2, 1, 64, 8, BF), ([1500], [200], (), 0.3, [], 7, 1, 128, 64, F16),
    ([900, 70], [64, 64], (), 0.05, [], 64, 8, 128, 16, BF), ([2100], [1024], (), 0.2, [], 1, 1, 64, 16, BF), ([2500], [2400], (), 0.1, [], 2, 1, 64, 32, BF),
    # prefixes: a group's members with trees and without, tokens not in use in front of shared pages
    ([400, 390, 380, 100], [3, 5, 7, 2], (2,), 0.2, [([2, 0, 1], 320)], 4, 1, 64, 32, F16),
    ([300, 200, 310, 250, 99], [9, 1, 30, 4, 8], (), 0.3, [([3, 0], 200), ([1, 4, 2], 80)], 28, 4, 128, 8, BF),
    ([2000 + i for i in range(20)], [4] * 20, (3, 5), 0.1, [(list(range(20)), 1984)], 32, 8, 128, 16, BF),
    ([700, 650, 300, 66], [90, 40, 0, 2], (0,), 0.0, [([0, 1, 2, 3], 64)], 7, 1, 128, 32, BF),
    ([5000], [25], (), 0.0, [], 32, 8, 128, 16, BF), ([5000, 4000], [31, 17], (), 0.1, [], 28, 4, 64, 32, F16),
    # several blocks of 256 rows
    ([3000, 1000, 2500, 64], [64, 40, 50, 60], (), 0.1, [], 64, 8, 128, 16, BF),
    ([3000, 2900], [64, 80], (), 0.1, [], 32, 4, 64, 64, F16), ([9000], [100], (), 0.0, [], 8, 1, 128, 16, BF),
    ([9000, 30, 8000], [40, 60, 64], (2,), 0.0, [], 16, 2, 128, 32, F16),
    # one row of bits that no token sets: none in use
    ([100, 200], [6, 3], (), 1.0, [], 4, 2, 128, 16, BF),
]


@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_trees(case, fixed):
    lens, new, chains, unused, prefixes, H, KVH, D, page, dtype = CASES[case]
    print(f"\n[case] tree attention {case} lens={lens[:6]} new={new[:6]} H={H} KVH={KVH} D={D} page={page} {dtype}",
          flush=True)
    r = random.Random(case)
    trees = [None if b in chains else random_tree(r, t, unused) for b, t in enumerate(new)]
    q, k, v, table, plan = _case(lens, new, trees, prefixes, H, KVH, D, page, dtype, case, fixed=fixed)
    want = _reference(q, k, v, table, lens, new, trees)
    few = sum(new) * H // KVH <= 16
    for rounded in (None, False, True):
        out = paged_attention(q, k, v, table, plan, rounded=rounded)
        _check(out, want, dtype, rounded=not few)
        assert torch.equal(out, paged_attention(q, k, v, table, plan, rounded=rounded))  # the same bits each time
    none = torch.tensor([not seen_tokens(n, t, p, i) for n, t, p in zip(lens, new, trees) for i in range(t)])
    assert (out[none.cuda()] == 0).all()


def test_chains_are_sequences():
    """A tree that is a chain has the plain plan's values; a batch in which no tree
    is a real one, its bits."""
    print("\n[case] chains as trees", flush=True)
    lens, new = [1000, 200, 64], [5, 40, 64]
    q, k, v, table, plan = _case(lens, new, [list(range(-1, t - 1)) for t in new], [], 8, 2, 128, 16, BF)
    plain = PagedPlan(lens, heads=8, kv_heads=2, new_tokens=new)
    assert torch.equal(plan.positions, plain.positions)
    assert torch.equal(paged_attention(q, k, v, table, plan), paged_attention(q, k, v, table, plain))


@pytest.mark.parametrize("H, KVH, D, dtype", [(2, 1, 128, BF), (4, 1, 64, F16), (8, 1, 128, F16), (16, 1, 64, BF),
                                              (32, 1, 128, BF)])
def test_masked_values_stay_out(H, KVH, D, dtype):
    """Infinities and NaN of drafted tokens, in K and V, reach those that follow
    them only, in every form of the kernel (4 to 512 rows)."""
    print(f"\n[case] masked values H={H} D={D} {dtype}", flush=True)
    r = random.Random(H)
    for rounded in (False, True):
        lens, new = [70, 135], [6, 16]
        trees = [[-1, 0, 0, 1, 1, 2], random_tree(r, 16, 0.2)]
        q, k, v, table, plan = _case(lens, new, trees, [], H, KVH, D, 8, dtype, H)
        base = _reference(q, k, v, table, lens, new, trees)
        v[table[0, 65 // 8].long(), 65 % 8], k[table[0, 65 // 8].long(), 65 % 8] = math.nan, math.inf
        v[table[0, 66 // 8].long(), 66 % 8] = -math.inf
        bad = 5
        v[table[1, (119 + bad) // 8].long(), (119 + bad) % 8] = math.inf
        out = paged_attention(q, k, v, table, plan, rounded=rounded)
        assert out[[1, 3, 4]].isnan().all() and (out[[2, 5]] == -math.inf).all()
        hit = torch.tensor([False, True, True, True, True, True]
                           + [119 + bad in seen_tokens(135, 16, trees[1], i) for i in range(16)]).cuda()
        assert (out[6:][hit[6:]] == math.inf).all()
        _check(out[~hit], tuple(x[~hit] for x in base), dtype)


def test_masked_values_beside_plain_sequences():
    """The same in a batch whose other sequence has no tree: later tokens stay out there."""
    print("\n[case] masked values beside a sequence without a tree", flush=True)
    for H, KVH, D in ((4, 2, 128), (16, 1, 64), (40, 1, 128)):
        lens, new, trees = [100, 140], [5, 30], [[-1, 0, 0, 1, 2], None]
        q, k, v, table, plan = _case(lens, new, trees, [], H, KVH, D, 16, BF, H)
        base = _reference(q, k, v, table, lens, new, trees)
        v[table[1, 130 // 16].long(), 130 % 16], k[table[1, 130 // 16].long(), 130 % 16] = math.inf, math.nan
        v[table[0, 98 // 16].long(), 98 % 16] = math.nan
        out = paged_attention(q, k, v, table, plan)
        hit = torch.tensor([False, False, False, True, False] + [110 + i >= 130 for i in range(30)]).cuda()
        assert not torch.isfinite(out[hit]).any()
        _check(out[~hit], tuple(x[~hit] for x in base), BF)


def test_tokens_not_in_use_behind_bad_prefixes():
    """Zeros of tokens not in use, also where the context holds infinities and NaN."""
    print("\n[case] not in use behind infinities", flush=True)
    lens, new, trees = [300, 290, 80], [4, 4, 4], [[-1, -2, 0, -2], [-2] * 4, [-1, -2, 0, 0]]
    for prefixes in ([], [([0, 1], 256)]):
        q, k, v, table, plan = _case(lens, new, trees, prefixes, 8, 2, 128, 16, BF)
        v[table[0, 3].long()], v[table[2, 0].long(), 2] = math.inf, math.nan
        v[table[1, 5].long()] = math.nan
        out = paged_attention(q, k, v, table, plan)
        zero = torch.tensor([1, 3, 4, 5, 6, 7, 9]).cuda()
        assert (out[zero] == 0).all() and not torch.isfinite(out[[0, 2]]).any() and out[[8, 10, 11]].isnan().all()


def test_large_scores():
    """Scores whose exponents need the maximum taken off before they are scaled."""
    print("\n[case] large scores", flush=True)
    lens, new, trees = [200, 90], [9, 5], [[-1, 0, 0, 1, 1, 2, 2, -1, 7], [-1, 0, 0, 1, 2]]
    q, k, v, table, plan = _case(lens, new, trees, [], 8, 2, 128, 16, BF)
    q = q * 300
    _check(paged_attention(q, k, v, table, plan), _reference(q, k, v, table, lens, new, trees), BF, rounded=True)


def test_replays_follow_other_trees():
    """A captured call, its plan updated to other lengths and trees between the
    replays, with the program's own work between them."""
    print("\n[case] replays", flush=True)
    r, new = random.Random(3), [16, 9, 16]
    lens = [300, 128, 511]
    trees = [random_tree(r, t, 0.1) for t in new]
    q, k, v, table, plan = _case([511] * 3, new, trees, [], 32, 8, 128, 16, BF, fixed=True)
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.5)
    plan.update(lens)
    paged_attention(q, k, v, table, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, k, v, table, plan)
    for lens, other in ((lens, None), ([64, 9, 130], [random_tree(r, t, 0.3) for t in new]), ([500, 0, 16], None),
                        ([511, 300, 3], [random_tree(r, t) for t in new])):
        plan.update(lens, other)
        trees = other or trees
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(q, k, v, table, plan))
        _check(out, _reference(q, k, v, table, lens, new, trees), BF)
        q.copy_(torch.randn_like(q))
    with pytest.raises(RuntimeError, match="exceeds the block table"):
        plan.update([100000, 1, 1])
