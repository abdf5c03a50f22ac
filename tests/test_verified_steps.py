"""Steps that verify drafted trees, stage by stage against float64, each stage on what
the one before really gave: tables, normed and rotated heads in the pages, attention of
every node, and the rows that stay, move and are copied.  Here on the CPU, and with
mistakes in the oracle that the bounds must not hold; tests/test_verified_steps_gpu.py
runs the same on the GPU."""
import math
import random

import pytest
import torch

from santa_amd.paged import PagedKVCache, paged_attention, rope_append, rope_tables
from test_draft_trees import path, random_tree
from test_tree_probabilities import tight
from test_verified_drafts_gpu import Layer

R = 32  # rotated dims


class Traced(Layer):
    """The layer, whose stages of the last step are kept."""

    def step(self, ids, cache, plan):
        dev = ids.device
        cos, sin = rope_tables(plan.positions, R, scaling=self.scaling, interleaved=True, dtype=self.dtype)
        q = rope_append(self.embed.to(dev)[ids], cos, sin, cache.k[0], cache.v[0], cache.block_table, plan,
                        q_norm=self.q_norm.to(dev), k_norm=self.k_norm.to(dev), interleaved=True)
        a = paged_attention(q, cache.k[0], cache.v[0], cache.block_table, plan)
        self.last = [t.cpu() for t in (cos, sin, q, a)]


def heads(layer, x, cos, sin):
    """Normed and rotated q and k heads of x [n, H + 2 KVH, D] in float64 and their
    bounds: as tests/test_rotary_gpu.py has them."""
    H, D = layer.H, layer.D
    y = x[:, :H + layer.KVH].double()
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6)
    y = y * torch.cat([layer.q_norm.double().expand(H, D), layer.k_norm.double()])
    a, b = y[..., :R:2].clone(), y[..., 1:R:2].clone()
    c, s = cos.double()[:, None, ::2], sin.double()[:, None, ::2]
    size = y.abs()
    size[..., :R:2], size[..., 1:R:2] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    y[..., :R:2], y[..., 1:R:2] = a * c - b * s, b * c + a * s
    half = torch.finfo(layer.dtype).eps / 2
    bound = (D / 2 + 10) * 2.0 ** -24 * size * (1 + half) + half * y.abs()
    return y, bound + 2.0 ** -25 if layer.dtype == torch.float16 else bound


def attend(layer, q, k, v):
    """A node's attention over rows k, v [n, KVH, D] in float64: values, mean of |v|,
    the scores' bound [H, D]."""
    D = layer.D
    kh, vh = (t.double().repeat_interleave(layer.H // layer.KVH, 1) for t in (k, v))
    p = torch.softmax((kh * q.double()).sum(-1) / math.sqrt(D), 0)[..., None]
    size = (kh * q.double()).abs().sum(-1).amax(0) / math.sqrt(D)
    return (p * vh).sum(0), (p * vh.abs()).sum(0), (2 * (D + 2) * 2.0 ** -24 * size + 2.0 ** -20)[:, None].expand(-1, D)


def checked_steps(dtype, device, mistake=None):
    """The steps with their stages checked; the share of its bound that each node's
    attention takes, for an oracle that makes the mistake."""
    layer, r = Traced(dtype, 1), random.Random(2)
    cache = PagedKVCache(1, 200, 16, kv_heads=2, head_dim=64, max_seqs=6, max_len=400, dtype=dtype, device=device)
    gone, *seqs = cache.add([50, 70, 20, 90])
    g = torch.Generator().manual_seed(3)
    rows = {}  # of each sequence: K and V of every place, as they were first written
    shares = []

    def stored(s, places):
        table = cache.block_table.cpu()
        return [tuple(pool[0].cpu()[int(table[s, p // 16]), p % 16].clone() for pool in (cache.k, cache.v)) for p in places]

    def as_written(s):
        return all(torch.equal(a, b) for x, y in zip(stored(s, range(len(rows[s]))), rows[s]) for a, b in zip(x, y))

    def check_heads(ids, at, depth, s, first, t):
        """Tokens at rows `at` of the step, at these positions, and what the pages
        hold at places first .. first + t - 1 of sequence s."""
        cos, sin, q, _ = (x[at] for x in layer.last)
        f, up = layer.scaling.frequencies(R, 10000.0)
        angle = (torch.tensor(depth, dtype=torch.float64)[:, None] * torch.tensor(f, dtype=torch.float64)).repeat_interleave(2, -1)
        half = torch.finfo(dtype).eps / 2
        for got, want in ((cos, angle.cos()), (sin, angle.sin())):
            assert ((got.double() - want).abs() <= half * want.abs() + 5 * 2.0 ** -24).all()
        x = layer.embed[ids]
        want, bound = heads(layer, x, cos, sin)
        kv = stored(s, range(first, first + t))
        got = torch.cat([q, torch.stack([k for k, _ in kv])], 1).double()
        assert ((got - want).abs() <= bound).all()
        assert torch.equal(torch.stack([v for _, v in kv]), x[:, layer.H + layer.KVH:])
        return kv

    new = cache.lengths(seqs)
    ids = torch.randint(0, layer.V, (sum(new),), generator=g)
    layer.step(ids.to(device), cache, cache.plan(seqs, 8, new))
    t0 = 0
    for s, n in zip(seqs, new):
        rows[s] = check_heads(ids[t0:t0 + n], list(range(t0, t0 + n)), list(range(n)), s, 0, n)
        t0 += n
    cache.free([gone])
    kids = cache.fork(seqs[2], 2)
    rows.update((s, list(rows[seqs[2]])) for s in kids)
    seqs += kids
    for step in range(4):
        new = [r.choice((1, 5, 16, 30)) for _ in seqs]
        at = cache.lengths(seqs)
        cache.extend(seqs, new)
        trees = [random_tree(r, t, 0.1) for t in new]
        ids = torch.randint(0, layer.V, (sum(new),), generator=g)
        layer.step(ids.to(device), cache, cache.plan(seqs, 8, new, parents=trees))
        t0, kept = 0, []
        for s, n, parents in zip(seqs, at, trees):
            assert len(rows[s]) == n and as_written(s)
            used = [i for i, p in enumerate(parents) if p != -2]
            depth = [n + len(path(parents, i)) - 1 for i in used]
            new_rows = dict(zip(used, [check_heads(ids[[t0 + i]], [t0 + i], [d], s, n + i, 1)[0] for i, d in zip(used, depth)]))
            _, _, q, a = layer.last
            for i, parent in enumerate(parents):
                if parent == -2:
                    assert (a[t0 + i] == 0).all()
                    continue
                seen = rows[s] + [new_rows[j] for j in path(parents, i)]
                others = [j for j in used if j not in path(parents, i)]
                if mistake == "a sibling" and others:
                    seen = seen + [new_rows[others[0]]]
                elif mistake == "a row":
                    seen = seen[:n - 1] + [seen[0]] + seen[n:]
                elif mistake == "a sibling":
                    continue
                k, v = (torch.stack(x) for x in zip(*seen))
                out = torch.zeros_like(a[t0 + i]) if mistake == "zeros" else a[t0 + i]
                shares.append(tight(out, attend(layer, q[t0 + i], k, v), dtype, len(seen), v.abs().max().item()))
            kept.append(path(parents, r.choice(used)) if used else [])
            rows[s] = rows[s] + [new_rows[j] for j in kept[-1]]
            t0 += len(parents)
        cache.keep(seqs, new, kept)
        if step == 1:
            assert cache.compact() == cache.used_pages
    assert all(as_written(s) for s in seqs) and cache.lengths(seqs) == [len(rows[s]) for s in seqs]
    return shares


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_steps(dtype):
    shares = checked_steps(dtype, "cpu")
    assert len(shares) > 150 and max(shares) <= 1


@pytest.mark.parametrize("mistake", ["zeros", "a sibling", "a row"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mistakes_do_not_pass(dtype, mistake):
    """Outputs of zeros, one token too many or one row in another's place are outside
    of the bound at every node."""
    assert min(checked_steps(dtype, "cpu", mistake)) > 1
