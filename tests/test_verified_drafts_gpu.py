"""A step that verifies drafted trees, its parts together on the GPU: rotary tables,
normed and rotated heads into pages, tree attention, rules on logits, accepted paths
kept, captured and not; and the model's trees.  Every case prints its name before
touching the GPU."""
import math
import random

import pytest
import torch

from santa_amd.logits import adjust_logits
from santa_amd.paged import PagedKVCache, PagedPlan, RopeScaling, paged_attention, rope_append, rope_tables
from santa_amd.runtime import LlamaShape, NHDCache, RandomLlama
from test_draft_trees import path, random_tree

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
SMALL = LlamaShape(hidden=1024, intermediate=2048, heads=8, kv_heads=2, layers=3, vocab=1000)


class Layer:
    """One attention layer with normed heads, half of them rotated in adjacent pairs
    at scaled positions, and a head, for sequences that a dictionary holds in float64."""

    H, KVH, D, V = 8, 2, 64, 331
    scaling = RopeScaling("llama3", 8.0, 64)

    def __init__(self, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.dtype = dtype
        self.embed = r(self.V, self.H + 2 * self.KVH, self.D).to(dtype)
        self.q_norm, self.k_norm = r(self.D).add(1).to(dtype), r(self.KVH, self.D).add(1).to(dtype)
        self.head = r(self.H * self.D, self.V).div(math.sqrt(self.H * self.D)).to(dtype)

    def step(self, ids, cache, plan):
        dev = ids.device
        cos, sin = rope_tables(plan.positions, 32, scaling=self.scaling, interleaved=True, dtype=self.dtype)
        q = rope_append(self.embed.to(dev)[ids], cos, sin, cache.k[0], cache.v[0], cache.block_table, plan,
                        q_norm=self.q_norm.to(dev), k_norm=self.k_norm.to(dev), interleaved=True)
        a = paged_attention(q, cache.k[0], cache.v[0], cache.block_table, plan)
        return a.view(len(ids), -1).float() @ self.head.to(dev).float()

    def exact(self, ids):
        """Logits behind the last of a sequence's tokens in float64, and how far
        roundings to 16 bits can move them: cos, sin and the rotated heads by eps of
        |x c| + |y s| each, so a score by the sum of what that makes of its products;
        a probability by twice the largest such move and its own rounding, the output
        by its rounding; a tenth more for the moves' products with one another."""
        eps = torch.finfo(self.dtype).eps / 2
        n = len(ids)
        x = self.embed[ids].double()
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        q = y[:, :self.H] * self.q_norm.double()
        k = y[:, self.H:self.H + self.KVH] * self.k_norm.double()
        f, _ = self.scaling.frequencies(32, 10000.0)
        angle = torch.arange(n, dtype=torch.float64)[:, None] * torch.tensor(f, dtype=torch.float64)
        off = []
        for t in (q, k):
            a, b = t[..., :32:2].clone(), t[..., 1:32:2].clone()
            c, s = angle.cos()[:, None], angle.sin()[:, None]
            size = 2 * t.abs()
            size[..., :32:2], size[..., 1:32:2] = 2 * ((a * c).abs() + (b * s).abs()), 2 * ((b * c).abs() + (a * s).abs())
            off.append(eps * size)
            t[..., :32:2], t[..., 1:32:2] = a * c - b * s, b * c + a * s
        k, k_off = (t.repeat_interleave(self.H // self.KVH, 1) for t in (k, off[1]))
        moved = torch.einsum("hd,nhd->hn", off[0][-1], k.abs()) + torch.einsum("hd,nhd->hn", q[-1].abs(), k_off)
        moved = torch.expm1(2 * moved.amax(-1) / math.sqrt(self.D))[:, None] + eps
        v = x[:, self.H + self.KVH:].repeat_interleave(self.H // self.KVH, 1)
        p = torch.softmax(torch.einsum("hd,nhd->hn", q[-1], k) / math.sqrt(self.D), -1)
        out, size = torch.einsum("hn,nhd->hd", p, v), torch.einsum("hn,nhd->hd", p, v.abs())
        head = self.head.double()
        return out.reshape(-1) @ head, 1.1 * (moved * size + eps * out.abs()).reshape(-1) @ head.abs() + 1e-5


@pytest.mark.parametrize("dtype", [BF, F16])
def test_steps(dtype):
    """Prompts, then trees, accepted paths and the next trees behind them: each node's
    logits are its whole path's, and the rules' those that its path has seen."""
    print(f"\n[case] steps {dtype}", flush=True)
    layer, r = Layer(dtype, 1), random.Random(2)
    cache = PagedKVCache(1, 200, 16, kv_heads=2, head_dim=64, max_seqs=6, max_len=400, dtype=dtype)
    gone, *seqs = cache.add([50, 70, 20, 90])
    tokens = torch.randint(0, layer.V, (6, 400), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    dev = tokens.cuda()
    layer.step(torch.cat([dev[s, :n] for s, n in zip(seqs, (70, 20, 90))]).long(), cache, cache.plan(seqs, 8, [70, 20, 90]))
    cache.free([gone])
    kids = cache.fork(seqs[2], 2)
    tokens[kids] = tokens[seqs[2]].clone()
    dev.copy_(tokens)
    seqs += kids
    prompts = torch.zeros(6, dtype=torch.int32)
    prompts[seqs] = torch.tensor(cache.lengths(seqs), dtype=torch.int32)
    for step in range(4):
        new = [r.choice((1, 5, 16, 30)) for _ in seqs]
        at = cache.lengths(seqs)
        cache.extend(seqs, new)
        trees = [random_tree(r, t, 0.1) for t in new]
        plan = cache.plan(seqs, 8, new, parents=trees)
        drafts = torch.randint(0, layer.V, (sum(new),), generator=torch.Generator().manual_seed(step))
        t0 = 0
        for s, n, t in zip(seqs, at, new):
            tokens[s, n:n + t] = drafts[t0:t0 + t]
            t0 += t
        dev.copy_(tokens)
        logits = layer.step(drafts.cuda(), cache, plan)
        ruled = adjust_logits(logits, dev, plan, prompts=prompts.cuda(), repetition=1.5, presence=0.3, frequency=0.1)
        chosen = adjust_logits(logits, dev, plan, prompts=prompts.cuda(), repetition=1.5, presence=0.3, frequency=0.1,
                               greedy=True).tolist()
        assert chosen == ruled.argmax(-1).tolist()
        t0, kept = 0, []
        for s, n, parents in zip(seqs, at, trees):
            used = [i for i, p in enumerate(parents) if p != -2]
            for i in used:
                ids = torch.cat([tokens[s, :n], tokens[s, n:][path(parents, i)]]).long()
                want, bound = layer.exact(ids)
                got = logits[t0 + i].double().cpu()
                assert ((got - want).abs() <= bound).all(), (step, s, i)
                count = torch.bincount(ids[int(prompts[s]):], minlength=layer.V)
                seen = torch.bincount(ids, minlength=layer.V) > 0
                y = torch.where(seen, torch.where(got > 0, got / 1.5, got * 1.5), got) - 0.1 * count - 0.3 * (count > 0)
                assert (ruled[t0 + i].double().cpu() - y).abs().max() <= 1e-5
            kept.append(path(parents, r.choice(used)) if used else [])
            t0 += len(parents)
        cache.keep(seqs, new, kept)
        for s, n, k in zip(seqs, at, kept):
            tokens[s, n:n + len(k)] = tokens[s, n:][k].clone()
        dev.copy_(tokens)
        if step == 1:
            assert cache.compact() == cache.used_pages
    assert cache.lengths(seqs) == [n + len(k) for n, k in zip(at, kept)]


def test_captured_step():
    """Tables, append, attention, rules and the chosen tokens in one graph, replayed
    over other lengths and trees, its cache kept between the replays."""
    print("\n[case] captured step", flush=True)
    layer, r = Layer(BF, 1), random.Random(5)
    for name in ("embed", "q_norm", "k_norm", "head"):
        setattr(layer, name, getattr(layer, name).cuda())
    cache = PagedKVCache(1, 100, 16, kv_heads=2, head_dim=64, max_seqs=3, max_len=300)
    seqs = cache.add([100, 30, 60])
    tokens = torch.randint(0, layer.V, (3, 304), device="cuda", dtype=torch.int32)
    layer.step(torch.cat([tokens[s, :n] for s, n in zip(seqs, (100, 30, 60))]).long(), cache, cache.plan(seqs, 8, [100, 30, 60]))
    new = [16, 9, 16]
    bits = torch.randint(-(1 << 31), 1 << 31, (41, 11), device="cuda").to(torch.int32)
    cache.extend(seqs, new)
    plan = PagedPlan([116, 39, 76], heads=8, kv_heads=2, new_tokens=new, rows=seqs, fixed=True,
                     parents=[random_tree(r, t) for t in new])
    ids = torch.randint(0, layer.V, (41,), device="cuda")

    def step(plan):
        logits = layer.step(ids, cache, plan)
        return logits, adjust_logits(logits, tokens, plan, repetition=1.2, allowed=bits, greedy=True)

    step(plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, token = step(plan)
    for i in range(4):
        trees = [random_tree(r, t, 0.1) for t in new]
        at = [n - t for n, t in zip(cache.lengths(seqs), new)]
        plan.update(cache.lengths(seqs), trees)
        ids.copy_(torch.randint(0, layer.V, (41,), device="cuda"))
        t0 = 0
        for s, n, t in zip(seqs, at, new):
            tokens[s, n:n + t] = ids[t0:t0 + t]
            t0 += t
        graph.replay()
        torch.cuda.synchronize()
        want, chosen = step(cache.plan(seqs, 8, new, parents=trees))
        assert torch.equal(logits, want) and torch.equal(token, chosen)
        kept, _ = plan.accepted(ids.tolist(), token.tolist()) if i % 2 else ([path(t, len(t) // 2) if t[len(t) // 2] > -2 else []
                                                                             for t in trees], None)
        cache.keep(seqs, new, kept)
        for s, n, k in zip(seqs, at, kept):
            tokens[s, n:n + len(k)] = tokens[s, n:][k].clone()
        cache.extend(seqs, new)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_model_trees(dtype):
    """The model's logits of drafted nodes are those of each node's path prefilled by
    itself, to the tolerance of the runtime's decode against its prefill, also behind
    paths that were kept."""
    print(f"\n[case] model trees {dtype}", flush=True)
    model = RandomLlama(SMALL, seed=11, std=0.05, device="cuda", dtype=dtype)
    g, r = torch.Generator().manual_seed(5), random.Random(4)
    cache = PagedKVCache(3, 200, 16, kv_heads=2, head_dim=128, max_seqs=4, max_len=500, dtype=dtype)
    first, = cache.add([0])
    texts = torch.randint(0, SMALL.vocab, (3, 200), generator=g).cuda()
    texts[1:] = texts[0]
    model.extend(texts[:1], cache, [first])
    seqs = [first, *cache.fork(first, 2)]
    texts = list(texts)
    for step in range(3):
        trees = [random_tree(r, t, 0.1) for t in (9, 1, 17)]
        new = [len(t) for t in trees]
        drafts = torch.randint(0, SMALL.vocab, (sum(new),), generator=g).cuda()
        logits = model.extend(drafts, cache, seqs, new, parents=trees)
        assert logits.shape == (sum(new), SMALL.vocab)
        t0, kept = 0, []
        for b, parents in enumerate(trees):
            used = [i for i, p in enumerate(parents) if p != -2]
            for i in used[::3] + used[-1:]:
                ids = torch.cat([texts[b], drafts[t0:][path(parents, i)]])
                want = model.prefill(ids[None], NHDCache(SMALL, 1, len(ids), dtype, "cuda"))[0]
                assert (logits[t0 + i] - want).abs().max() <= 0.05 * want.abs().max()
            kept.append(path(parents, used[-1]) if used else [])
            texts[b] = torch.cat([texts[b], drafts[t0:][kept[-1]]])
            t0 += len(parents)
        cache.keep(seqs, new, kept)
        assert cache.lengths(seqs) == [len(t) for t in texts]
