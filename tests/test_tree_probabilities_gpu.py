"""Probabilities of drafted trees on the GPU: in two parts, whatever is beside the
tree, in every form of the kernel.

Tolerance (tests/test_paged_probabilities_gpu.py): the output is rounded once, eps of
its value; a probability's second part, at most two steps of the first, is rounded
(4 eps^2 of the mean of |v|), or is less than half of the smallest number, 2^-25 of a
reference of 2^7, in f16; float32 scores.

Every case prints its name before touching the GPU.
"""
import math
import random

import pytest
import torch

from santa_amd.paged import PagedPlan, paged_attention
from test_draft_trees import random_tree, seen_tokens
from test_draft_trees_gpu import _case, _reference
from test_shared_pages_gpu import _check
from test_tree_probabilities import branching, chain, tight

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16

# rows of a tree's pass: 17 to 32, 64, 128, 256, several blocks, with and without a prefix
CASES = [
    # lens, new, sequences without a tree, prefixes, H, KVH, D, page, dtype
    ([500], [6], (), [], 32, 8, 128, 16, BF), ([70, 64, 200], [7, 5, 8], (), [], 8, 2, 64, 8, F16),
    ([1500, 300], [16, 13], (), [], 16, 4, 128, 32, BF), ([1500, 90], [16, 16], (), [], 4, 1, 64, 16, F16),
    ([900, 70], [25, 32], (), [], 32, 8, 128, 16, F16), ([2000], [128], (), [], 1, 1, 64, 8, BF),
    ([1300, 129], [64, 33], (), [], 8, 2, 128, 64, BF), ([2500], [256], (), [], 2, 2, 64, 16, F16),
    ([3000, 1000], [64, 90], (), [], 64, 8, 128, 16, BF), ([4000], [64], (), [], 64, 8, 128, 16, F16),
    ([400, 390, 380, 100], [30, 5, 7, 2], (), [([2, 0, 1], 256)], 4, 1, 64, 32, F16),
    ([2000 + i for i in range(12)], [4] * 12, (), [(list(range(12)), 1920)], 32, 8, 128, 16, BF),
    # beside prefills and decoded tokens
    ([500, 900], [6, 300], (1,), [], 32, 8, 128, 16, BF), ([300, 700, 65, 80], [16, 90, 1, 9], (1, 2), [], 16, 4, 64, 8, F16),
    ([900, 850, 870, 30], [64, 300, 40, 1], (1, 3), [([0, 1, 2], 512)], 8, 1, 128, 16, BF),
    ([400, 390, 380, 395], [7, 9, 12, 2], (1, 3), [([0, 1, 2, 3], 320)], 28, 4, 64, 32, F16),
    ([2000 + i for i in range(12)], [12, 40, 1] * 4, (1, 2, 4, 5, 7, 8, 10, 11), [(list(range(12)), 1920)], 8, 2, 128, 64, BF),
]


def _rows(new, which):
    return torch.tensor([which(b) for b, t in enumerate(new) for _ in range(t)])


@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_trees_are_not_rounded(case, fixed):
    lens, new, chains, prefixes, H, KVH, D, page, dtype = CASES[case]
    print(f"\n[case] tree probabilities {case} lens={lens[:6]} new={new[:6]} H={H} KVH={KVH} D={D} {dtype}", flush=True)
    r = random.Random(case)
    trees = [None if b in chains else random_tree(r, t, 0.1) if t > 5 else branching(t) for b, t in enumerate(new)]
    q, k, v, table, plan = _case(lens, new, trees, prefixes, H, KVH, D, page, dtype, case, fixed=fixed)
    want = _reference(q, k, v, table, lens, new, trees)
    top = v.nan_to_num(0.0).abs().max().item()
    out = paged_attention(q, k, v, table, plan)
    tree = _rows(new, lambda b: b not in chains).cuda()
    assert tight(out[tree], [x[tree] for x in want], dtype, max(lens), top) <= 1
    _check(out, want, dtype)
    assert torch.equal(out, paged_attention(q, k, v, table, plan))
    exact = paged_attention(q, k, v, table, plan, rounded=False)
    assert tight(exact, want, dtype, max(lens), top) <= 1
    if not chains:
        assert torch.equal(out, exact)
    _check(paged_attention(q, k, v, table, plan, rounded=True), want, dtype)


@pytest.mark.parametrize("H, KVH, D, dtype", [(2, 1, 128, BF), (4, 1, 64, F16), (8, 1, 128, F16), (16, 1, 64, BF),
                                              (32, 1, 128, BF), (32, 1, 128, F16)])
@pytest.mark.parametrize("beside", [1, 40])
def test_masked_values_in_two_parts(H, KVH, D, dtype, beside):
    """Infinities and NaN of drafted tokens reach those that follow them only, and
    leave the others what they were; beside a sequence without a tree, rounded or not."""
    print(f"\n[case] masked values in two parts H={H} D={D} beside={beside} {dtype}", flush=True)
    r = random.Random(H)
    lens, new = [70, 135, 99], [6, 16, beside]
    trees = [[-1, 0, 0, 1, 1, 2], random_tree(r, 16, 0.2), None]
    q, k, v, table, plan = _case(lens, new, trees, [], H, KVH, D, 8, dtype, H)
    base = _reference(q, k, v, table, lens, new, trees)
    top = v.nan_to_num(0.0).abs().max().item()
    clean = paged_attention(q, k, v, table, plan)
    v[table[0, 65 // 8].long(), 65 % 8], k[table[0, 65 // 8].long(), 65 % 8] = math.nan, math.inf
    v[table[0, 66 // 8].long(), 66 % 8] = -math.inf
    v[table[1, (119 + 5) // 8].long(), (119 + 5) % 8] = math.inf
    hit = torch.tensor([False, True, True, True, True, True] + [124 in seen_tokens(135, 16, trees[1], i) for i in range(16)]
                       + [False] * beside).cuda()
    for rounded in (None, False):
        out = paged_attention(q, k, v, table, plan, rounded=rounded)
        assert out[[1, 3, 4]].isnan().all() and (out[[2, 5]] == -math.inf).all() and (out[6:22][hit[6:22]] == math.inf).all()
        ok = ~hit
        if rounded is None:
            ok[22:] = False
            assert torch.equal(out[22:], clean[22:])
        assert tight(out[ok], [x[ok] for x in base], dtype, max(lens), top) <= 1


def test_chains_beside_a_prefill():
    """Chains keep the bits of a plan without trees, whatever else is in the batch."""
    print("\n[case] chains beside a prefill", flush=True)
    lens, new = [1000, 200, 640, 64], [5, 40, 300, 64]
    for dtype in (BF, F16):
        q, k, v, table, plan = _case(lens, new, [chain(5), chain(40), None, chain(64)], [], 8, 2, 128, 16, dtype)
        plain = PagedPlan(lens, heads=8, kv_heads=2, new_tokens=new)
        assert torch.equal(paged_attention(q, k, v, table, plan), paged_attention(q, k, v, table, plain))


def test_replays_change_forms():
    """A captured call whose plan's trees are chains, and are not: the replays hold
    probabilities as the items say."""
    print("\n[case] replays that change forms", flush=True)
    lens, new, r = [300, 128, 511], [16, 9, 16], random.Random(3)
    q, k, v, table, plan = _case(lens, new, [chain(t) for t in new], [], 32, 8, 128, 16, BF, fixed=True)
    plain = PagedPlan(lens, heads=32, kv_heads=8, new_tokens=new, fixed=True)
    top = v.nan_to_num(0.0).abs().max().item()
    paged_attention(q, k, v, table, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, k, v, table, plan)
    for trees in ([chain(t) for t in new], [random_tree(r, t, 0.1) for t in new], [chain(16), branching(9), branching(16)],
                  [chain(t) for t in new]):
        plan.update(lens, trees)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(q, k, v, table, plan))
        tree = _rows(new, lambda b: trees[b] != chain(new[b])).cuda()
        want = _reference(q, k, v, table, lens, new, trees)
        if tree.any():
            assert tight(out[tree], [x[tree] for x in want], BF, max(lens), top) <= 1
        else:
            assert torch.equal(out, paged_attention(q, k, v, table, plain))
        q.copy_(torch.randn_like(q))
