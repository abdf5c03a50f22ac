"""A step that verifies drafted trees, its parts together, on the CPU: the model's
trees, rules on their logits, the accepted paths and what stays in the cache, against
decoding token by token."""
import random

import pytest
import torch

from santa_amd.logits import adjust_logits
from santa_amd.paged import PagedPlan
from santa_amd.runtime import ExactDecodeBackend, NHDCache, RandomLlama
from test_draft_trees import path, random_tree
from test_paged import TINY, _model_cache

RULES = dict(repetition=1.3, frequency=0.2, presence=0.1)


def prompts_and_table(model, cache, g, lens):
    seqs = cache.add([0] * len(lens))
    tokens = torch.zeros(cache.max_seqs, 120, dtype=torch.int32)
    for s, n in zip(seqs, lens):
        tokens[s, :n] = torch.randint(0, TINY.vocab, (n,), generator=g)
    logits = model.extend(torch.cat([tokens[s, :n] for s, n in zip(seqs, lens)]).long().to(model.device), cache, seqs, lens)
    return seqs, tokens.to(model.device), logits


def greedy(model, lens, steps, seed):
    """Token by token under the rules: [steps + 1] tokens of each sequence."""
    cache = _model_cache(TINY, dtype=model.dtype, device=model.device)
    g = torch.Generator().manual_seed(seed)
    seqs, tokens, logits = prompts_and_table(model, cache, g, lens)
    prompts = torch.zeros(cache.max_seqs, dtype=torch.int32)
    prompts[seqs] = torch.tensor(lens, dtype=torch.int32)
    prompts, out, at = prompts.to(model.device), [[] for _ in lens], list(lens)
    for i in range(steps + 1):
        plan = PagedPlan(at, heads=1, kv_heads=1, rows=seqs, device=model.device)
        chosen = adjust_logits(logits, tokens, plan, prompts=prompts, greedy=True, **RULES).tolist()
        for j, s in enumerate(seqs):
            out[j].append(chosen[j])
            tokens[s, at[j]] = chosen[j]
            at[j] += 1
        if i < steps:
            logits = model.extend(torch.tensor([[c] for c in chosen]).to(model.device), cache, seqs)
    return out


def drafted(r, truth, done, t):
    """A tree of t tokens whose first is the sequence's next one: the true
    continuation on one path up to somewhere, other tokens elsewhere."""
    parents = random_tree(r, t)
    parents[0] = -1
    parents = [p if i == 0 or p >= 0 else 0 for i, p in enumerate(parents)]
    drafts = [r.randrange(TINY.vocab) for _ in range(t)]
    good = path(parents, r.randrange(t))[:r.randint(1, t)]
    for depth, i in enumerate(good):
        if done + depth < len(truth):
            drafts[i] = truth[done + depth]
    drafts[0] = truth[done]
    return parents, drafts


def test_drafts_decode_the_same_tokens():
    """Trees of any shape decode what single tokens decode, in fewer steps."""
    model = RandomLlama(TINY, seed=3, std=0.08, dtype=torch.float32, device="cpu")
    lens, total = [20, 7, 33], 24
    truth = greedy(model, lens, total + 12, 5)
    cache = _model_cache(TINY)
    g, r = torch.Generator().manual_seed(5), random.Random(0)
    seqs, tokens, logits = prompts_and_table(model, cache, g, lens)
    prompts = torch.zeros(cache.max_seqs, dtype=torch.int32)
    prompts[seqs] = torch.tensor(lens, dtype=torch.int32)
    chosen = adjust_logits(logits, tokens, PagedPlan(lens, heads=1, kv_heads=1, rows=seqs, device="cpu"), prompts=prompts,
                           greedy=True, **RULES).tolist()
    out, steps = [[c] for c in chosen], 0
    while min(map(len, out)) <= total:
        order = r.sample(range(3), 3)
        trees = [drafted(r, truth[j], len(out[j]) - 1, r.choice((1, 5, 9))) for j in order]
        new, ids = [len(p) for p, _ in trees], [seqs[j] for j in order]
        at = cache.lengths(ids)
        for s, n, (p, d) in zip(ids, at, trees):
            tokens[s, n:n + len(d)] = torch.tensor(d, dtype=torch.int32)
        flat = [x for _, d in trees for x in d]
        logits = model.extend(torch.tensor(flat), cache, ids, new, parents=[p for p, _ in trees])
        assert logits.shape == (sum(new), TINY.vocab)
        plan = cache.plan(ids, TINY.heads, new, parents=[p for p, _ in trees])
        chosen = adjust_logits(logits, tokens, plan, prompts=prompts, greedy=True, **RULES)
        kept, following = plan.accepted(flat, chosen.tolist())
        cache.keep(ids, new, kept)
        for j, s, n, (p, d), k, c in zip(order, ids, at, trees, kept, following):
            tokens[s, n:n + len(k)] = torch.tensor([d[i] for i in k], dtype=torch.int32)
            out[j] += [d[i] for i in k[1:]] + [c]
            assert out[j] == truth[j][:len(out[j])], (steps, j)
        steps += 1
    assert steps < 0.8 * total and cache.lengths(seqs) == [n + len(o) - 1 for n, o in zip(lens, out)]


def test_tree_logits_are_those_of_their_paths():
    model = RandomLlama(TINY, seed=3, std=0.08, dtype=torch.float32, device="cpu")
    cache, g, r = _model_cache(TINY), torch.Generator().manual_seed(1), random.Random(1)
    seqs, tokens, _ = prompts_and_table(model, cache, g, [20, 9])
    trees = [random_tree(r, 7, 0.2), random_tree(r, 5)]
    drafts = torch.randint(0, TINY.vocab, (12,), generator=g)
    logits = model.extend(drafts, cache, seqs, [7, 5], parents=trees)
    t0 = 0
    for s, n, parents in zip(seqs, (20, 9), trees):
        for i, p in enumerate(parents):
            if p != -2:
                whole = torch.cat([tokens[s, :n].long(), drafts[t0:][path(parents, i)]])
                want = model.prefill(whole[None], NHDCache(TINY, 1, len(whole), torch.float32, "cpu"))[0]
                assert (logits[t0 + i] - want).abs().max() < 1e-5
        t0 += len(parents)


def test_accepted():
    parents = [[-1, 0, 0, 1, 2], [-1], [-2, -1], [-1, 0, 0], [-1, 0]]
    plan = PagedPlan([9, 5, 6, 2, 4], heads=1, kv_heads=1, new_tokens=[5, 1, 2, 3, 2], parents=parents, device="cpu")
    drafts = [4, 5, 6, 7, 8, 1, 0, 3, 9, 9, 9, 2, 2]
    chosen = [6, 0, 8, 0, 3, 7, 0, 0, 9, 9, 9, 5, 1]
    assert plan.accepted(drafts, chosen) == ([[0, 2, 4], [0], [], [], [0]], [3, 7, -1, -1, 5])
    for bad in (lambda: plan.accepted(drafts[:-1], chosen), lambda: plan.accepted(drafts, chosen + [1]),
                lambda: plan.accepted(drafts, [0.5] * 13),
                lambda: PagedPlan([5], heads=1, kv_heads=1, device="cpu").accepted([1], [1])):
        with pytest.raises(ValueError):
            bad()


def test_refused_trees_leave_the_sequences():
    model = RandomLlama(TINY, seed=3, std=0.08, dtype=torch.float32, device="cpu")
    cache = _model_cache(TINY)
    a, = cache.add([5])
    for parents, error in (([[0, 0]], RuntimeError), ([[-1]], ValueError), ([[-1, 0], [-1]], ValueError)):
        with pytest.raises(error):
            model.extend(torch.zeros(1, 2, dtype=torch.long), cache, [a], parents=parents)
        assert cache.lengths([a]) == [5] and cache.used_pages == 1
    with pytest.raises(ValueError, match="one new token"):
        model.extend(torch.zeros(1, 2, dtype=torch.long), cache, [a], parents=[[-1, 0]], backend=ExactDecodeBackend())
    with pytest.raises(ValueError, match="no trees"):
        model.extend(torch.zeros(1, 1, dtype=torch.long), cache, [a], parents=[[-1]], backend=ExactDecodeBackend())
    assert cache.lengths([a]) == [5]
