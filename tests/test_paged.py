"""Shared paged caches on the CPU: the host bookkeeping against a plain model of
it, the attention plan carried out in Python as the kernels carry it out, the
torch expressions, and refusals.  The bookkeeping and the planner are the
library's; nothing here needs a GPU.
"""
import ctypes
import math
import random

import pytest
import torch

from santa_amd import paged
from santa_amd.paged import PagedKVCache, PagedPlan, copy_pages, paged_attention, rope_append
from santa_amd.runtime import ExactDecodeBackend, LlamaShape, NHDCache, RandomLlama


class Model:
    """What the bookkeeping does, in the plainest form."""

    def __init__(self, pages, page, seqs):
        self.refs, self.page, self.rows = [0] * pages, page, [None] * seqs
        self.lens = [None] * seqs

    def free_rows(self):
        return [i for i, r in enumerate(self.rows) if r is None]

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def add(self, lengths):
        out = self.free_rows()[:len(lengths)]
        for s in out:
            self.rows[s], self.lens[s] = [], 0
        self.extend(out, lengths)
        return out

    def extend(self, seqs, tokens):
        for s, t in zip(seqs, tokens):
            if t and self.lens[s] % self.page and self.refs[self.rows[s][-1]] > 1:
                self.refs[self.rows[s][-1]] -= 1
                self.rows[s][-1] = self.take()
            self.lens[s] += t
            while len(self.rows[s]) * self.page < self.lens[s]:
                self.rows[s].append(self.take())

    def fork(self, s, n):
        out = self.free_rows()[:n]
        for c in out:
            self.rows[c], self.lens[c] = list(self.rows[s]), self.lens[s]
            for p in self.rows[s]:
                self.refs[p] += 1
        return out

    def free(self, seqs):
        for s in seqs:
            for p in self.rows[s]:
                self.refs[p] -= 1
            self.rows[s] = self.lens[s] = None

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        high = [p for p in range(n, len(self.refs)) if self.refs[p]]
        to = dict(zip(high, [p for p in range(n) if not self.refs[p]]))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [r and [to.get(p, p) for p in r] for r in self.rows]
        return n


def _cache(pages=40, page=8, seqs=9, max_len=100, layers=2, device="cpu"):
    return PagedKVCache(layers, pages, page, kv_heads=1, head_dim=16, max_seqs=seqs, max_len=max_len, dtype=torch.float32,
                        device=device)


def _write(cache, seq, lo, hi, value):
    """Tokens lo .. hi - 1 of a sequence hold value + their position."""
    for n in range(lo, hi):
        p, r = cache.pages(seq)[n // cache.page_size], n % cache.page_size
        for j, t in enumerate((*cache.k, *cache.v)):
            t[p, r] = value + n + 1000.0 * j


def _contents(cache, seq):
    n = cache.lengths([seq])[0]
    at = torch.arange(n)
    rows = cache.block_table[seq].cpu()[at // cache.page_size].long() if n else at
    return [t.cpu()[rows, at % cache.page_size, 0, 0].tolist() for t in (*cache.k, *cache.v)]


@pytest.mark.parametrize("seed", range(6))
def test_bookkeeping(seed):
    """Random operations: rows, references, the block table and every token's
    contents are those of the plain model; a refused one changes nothing."""
    r = random.Random(seed)
    cache, m = _cache(), Model(40, 8, 9)
    tokens = {}  # seq -> the value written at each position
    refused = 0
    for step in range(250):
        alive = [s for s, row in enumerate(m.rows) if row is not None]
        op = r.choice(("add", "extend", "extend", "fork", "free", "compact"))
        before = ([list(x) if x is not None else None for x in m.rows], list(m.refs), cache.block_table.clone())
        try:
            if op == "add":
                want = [r.choice((0, 1, 7, 8, 9, 30)) for _ in range(r.randint(0, 3))]
                seqs = cache.add(want)
                assert seqs == m.add(want)
                for s, n in zip(seqs, want):
                    tokens[s] = [10000.0 * step + i for i in range(n)]
                    _write(cache, s, 0, n, 10000.0 * step)
            elif op == "extend" and alive:
                seqs = r.sample(alive, r.randint(1, len(alive)))
                more = [r.choice((0, 1, 1, 5, 20)) for _ in seqs]
                had = cache.lengths(seqs)
                cache.extend(seqs, more)
                m.extend(seqs, more)
                for s, n, t in zip(seqs, had, more):
                    tokens[s] = tokens[s] + [10000.0 * step + n + i for i in range(t)]
                    _write(cache, s, n, n + t, 10000.0 * step)
            elif op == "fork" and alive:
                s, n = r.choice(alive), r.randint(0, 3)
                out = cache.fork(s, n)
                assert out == m.fork(s, n)
                tokens.update((c, list(tokens[s])) for c in out)
            elif op == "free" and alive:
                seqs = r.sample(alive, r.randint(1, len(alive)))
                cache.free(seqs)
                m.free(seqs)
            elif op == "compact":
                assert cache.compact() == m.compact()
        except RuntimeError as e:
            refused += 1
            assert "out of" in str(e) or "would hold" in str(e)
            assert torch.equal(cache.block_table, before[2])
        assert cache.used_pages == sum(x > 0 for x in m.refs)
        for s, row in enumerate(m.rows):
            if row is not None:
                assert cache.pages(s) == row and cache.lengths([s]) == [m.lens[s]]
                assert cache.block_table[s, :len(row)].tolist() == row
                assert _contents(cache, s) == [[v + 1000.0 * j for v in tokens[s]] for j in range(4)]
    assert refused > 0


def test_bookkeeping_refusals():
    cache = _cache()
    a, b = cache.add([10, 3])
    state = (cache.block_table.clone(), cache.used_pages, cache.pages(a), cache.pages(b))
    for call, text in [
        (lambda: cache.add([-1]), "at least 0"), (lambda: cache.add([105]), "has room for 104"),
        (lambda: cache.add([100] * 4), "out of pages"), (lambda: cache.add([1] * 8), "out of sequences"),
        (lambda: cache.extend([a, a], 1), "named twice"), (lambda: cache.extend([a, 7], 1), "no sequence 7"),
        (lambda: cache.extend([-1], 1), "no sequence -1"), (lambda: cache.extend([b, a], [1, -1]), "at least 0"),
        (lambda: cache.extend([b, a], [5, 100]), "would hold 110"), (lambda: cache.fork(5, 1), "no sequence 5"),
        (lambda: cache.fork(a, 8), "out of sequences"), (lambda: cache.free([a, 8]), "no sequence 8"),
        (lambda: cache.free([b, b]), "named twice"), (lambda: cache.lengths([3]), "no sequence 3"),
        (lambda: cache.tables([4]), "no sequence 4"), (lambda: cache.pages(2), "no sequence 2"),
        (lambda: cache.plan([a, 6], 2), "no sequence 6"), (lambda: cache.extend([a], [2 ** 31 - 1]), "would hold"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()
    for call in (lambda: cache.extend([a], [1, 2]), lambda: cache.extend([a], [1 << 31]), lambda: cache.fork(a, -1),
                 lambda: cache.add(3), lambda: cache.plan([a], 2, [1, 1])):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(cache.block_table, state[0]) and cache.used_pages == state[1]
    assert (cache.pages(a), cache.pages(b)) == state[2:]
    for args in ((0, 8, 4, 8), (4, 12, 4, 8), (4, 4, 4, 8), (4, 8, 0, 8), (4, 1 << 21, 4, 8)):
        with pytest.raises((RuntimeError, ValueError)):
            _cache(*args)
    # refused forks of a copied tail leave the references as they were
    full = _cache(pages=3, seqs=4)
    s, = full.add([20])
    kids = full.fork(s, 2)
    with pytest.raises(RuntimeError, match="out of pages: 2 needed, 0 free"):
        full.extend([s, *kids], 1)
    full.free(kids)
    full.extend([s], 1)  # alone again: no copy needed
    assert full.pages(s) == [0, 1, 2] and full.lengths([s]) == [21]


def test_last_holder_writes_in_place():
    cache = _cache()
    s, = cache.add([12])
    _write(cache, s, 0, 12, 5.0)
    kids = cache.fork(s, 2)
    cache.extend([*kids, s], 1)
    assert cache.pages(s) == [0, 1] and [cache.pages(k) for k in kids] == [[0, 2], [0, 3]]
    assert all([x[:12] for x in _contents(cache, k)] == [x[:12] for x in _contents(cache, s)] for k in kids)


def test_tables():
    cache = _cache()
    seqs = cache.add([9, 20, 3, 17])
    assert torch.equal(cache.tables(seqs), cache.block_table[:4])
    assert torch.equal(cache.tables([3, 0]), cache.block_table[[3, 0]])
    assert cache.tables([]).shape == (0, 13)


def test_copy_pages():
    g = torch.Generator().manual_seed(1)
    a, b = torch.randn(7, 8, 2, generator=g), torch.randn(7, 3, generator=g)
    view = torch.randn(7, 2, 5, generator=g)[:, 1]
    want = [t.clone() for t in (a, b, view)]
    for t in want:
        t[[0, 3, 2]] = t[[5, 5, 6]]
    copy_pages([a, b, view], [5, 5, 6], torch.tensor([0, 3, 2]))
    assert all(torch.equal(x, y) for x, y in zip((a, b, view), want))
    copy_pages(a, [], [])
    copy_pages([], [1], [2])
    for src, dst, text in [([0], [7], "no page 7"), ([-1], [0], "no page -1"), ([0, 1], [2, 2], "written twice"),
                           ([0, 1], [1, 2], "both read and written"), ([3], [3], "both read and written")]:
        with pytest.raises(RuntimeError, match=text):
            copy_pages(a, src, dst)
    for bad in (lambda: copy_pages(a, [0], [1, 2]), lambda: copy_pages([a, a[:5]], [0], [1]),
                lambda: copy_pages(a.transpose(1, 2), [0], [1]), lambda: copy_pages(a[:1].expand(7, 8, 2), [0], [1]),
                lambda: copy_pages(torch.zeros(5), [0], [1]), lambda: copy_pages(a, 0, 1)):
        with pytest.raises(ValueError):
            bad()
    assert torch.equal(a, want[0])


# --------------------------------------------------------------------- plan
def _shared_pools(lens, prefixes, page, KVH, D, seed, dtype=torch.float64, slack=3, spare=2):
    """Pools in random page order and the block table of sequences that share
    prefixes page by page (and only whole pages); unused entries name pages of
    NaN."""
    g = torch.Generator().manual_seed(seed)
    first = {b: (i, n // page) for i, (m, n) in enumerate(prefixes) for b in m}
    need = sum(n // page for _, n in prefixes) + sum(-(-n // page) - first.get(b, (0, 0))[1] for b, n in enumerate(lens))
    order = torch.randperm(need + spare, generator=g).tolist()
    bad, order = order[:spare], order[spare:]
    shared = [[order.pop() for _ in range(n // page)] for _, n in prefixes]
    table = torch.full((len(lens), max(1, -(-max(lens, default=0) // page) + slack)), bad[0], dtype=torch.int32)
    for b, n in enumerate(lens):
        row = list(shared[first[b][0]]) if b in first else []
        row += [order.pop() for _ in range(-(-n // page) - len(row))]
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    k, v = (torch.randn(need + spare, page, KVH, D, generator=g, dtype=torch.float32).to(dtype) for _ in range(2))
    k[bad], v[bad] = math.nan, math.nan
    for b, n in enumerate(lens):  # past the last token of the last page
        if n % page:
            k[table[b, n // page], n % page:] = math.nan
            v[table[b, n // page], n % page:] = math.nan
    return k, v, table


def _formula(q, k, v, table, lens, new, scale=None):
    """Token by token in float64."""
    N, H, D = q.shape
    page, KVH = k.shape[1:3]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, t0 = torch.zeros(N, H, D, dtype=torch.float64), 0
    for b, (n, t) in enumerate(zip(lens, new)):
        at = torch.arange(n)
        ks, vs = (x.cpu()[table.cpu()[b, at // page].long(), at % page].double() for x in (k, v))
        for i in range(max(0, t - n), t):
            m = n - t + i + 1
            for h in range(H):
                p = torch.softmax(ks[:m, h // (H // KVH)] @ q[t0 + i, h].double().cpu() * scale, 0)
                out[t0 + i, h] = p @ vs[:m, h // (H // KVH)]
        t0 += t
    return out


def _carry_out(q, k, v, table, plan):
    """The plan as the kernels carry it out: every item's parts, then the join."""
    info, data = plan._info, plan._data
    H, KVH = plan.heads, plan.kv_heads
    GH, page, D = H // KVH, k.shape[1], q.shape[2]
    N = plan.tokens
    out = torch.full((N, H, D), math.nan, dtype=torch.float64)
    part = {}
    written = set()
    items, seen = [], set()
    for w in range(info.groups):
        while w >= 0:
            assert w < info.items and w not in seen
            seen.add(w)
            items.append(data[16 * w:16 * w + 9].tolist())
            w = items[-1][8]
    for flags, row, begin, end, tok0, rows, pos0, base, _ in items:
        if rows == 0:
            continue
        assert begin % 64 == 0 and begin <= end and 0 < rows <= 256 and rows % GH == 0
        at = torch.arange(begin, end)
        kk, vv = (x[table[row, at // page].long(), at % page] for x in (k, v))
        for kv in range(KVH):
            for r in range(rows):
                tok = int(data[info.list_at + tok0 + r // GH]) if flags & 1 else tok0 + r // GH
                h = kv * GH + r % GH
                seen = at <= pos0 + r // GH
                s = (kk[:, kv] @ q[tok, h] / math.sqrt(D))[seen]
                m = s.max() if len(s) else torch.tensor(-3.4e38, dtype=torch.float64)
                e = torch.exp(s - m)
                res = (m, e.sum(), e @ vv[seen, kv])
                if flags & 2:
                    assert (tok, h) not in written
                    written.add((tok, h))
                    out[tok, h] = res[2] / res[1] if pos0 + r // GH >= 0 else 0.0
                else:
                    rec = base + kv * rows + r
                    assert rec not in part and rec < info.records
                    part[rec] = res
    for j in range(info.merge_tokens):
        tok = int(data[info.merge_at + j])
        if tok < 0:
            continue
        a, b = data[info.parts_at + 8 * tok:info.parts_at + 8 * tok + 8].view(2, 4).tolist()
        if b[3] == 0:
            continue
        for h in range(H):
            recs = [p[0] + (s * KVH + h // GH) * p[1] + p[2] + h % GH for p in (a, b) for s in range(p[3])]
            ps = [part.pop(x) for x in recs]
            top = max(p[0] for p in ps)
            w = [torch.exp(p[0] - top) for p in ps]
            assert (tok, h) not in written
            written.add((tok, h))
            pos = int(data[info.pos_at + 2 * tok])
            out[tok, h] = sum(x * p[2] for x, p in zip(w, ps)) / sum(x * p[1] for x, p in zip(w, ps)) if pos >= 0 else 0.0
    assert not part and len(written) == N * H
    return out


PLANS = [
    # lens, new tokens, prefixes, H, KVH, page
    ([1], [1], [], 4, 2, 8),
    ([0, 5, 64, 65], [1, 1, 1, 1], [], 2, 2, 8),
    ([130, 131, 200], [1, 1, 1], [([0, 1, 2], 128)], 4, 1, 16),
    ([130, 131, 200, 90], [1, 1, 1, 1], [([2, 0], 120), ([3, 1], 64)], 6, 2, 8),
    ([300, 20, 2, 0], [5, 20, 7, 3], [], 4, 2, 8),
    ([300, 310, 290, 70], [40, 33, 1, 0], [([0, 1, 2, 3], 64)], 7, 1, 32),
    ([200, 200, 200], [0, 1, 3], [([0, 1, 2], 190)], 2, 1, 8),
    ([], [], [], 4, 2, 8),
    ([90, 90], [1, 1], [([0, 1], 63)], 2, 1, 8),
    ([5000], [1], [], 2, 2, 64),
    ([700, 3], [300, 2], [], 8, 2, 16),
    ([260], [2], [], 128, 1, 64),
    ([100], [3], [], 256, 1, 8),
]


@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("case", range(len(PLANS)))
def test_plan(case, fixed):
    """Carried out item by item, a plan gives the formula's values: every token
    and head once, every part joined once, nothing read that is not a token."""
    lens, new, prefixes, H, KVH, page = PLANS[case]
    k, v, table = _shared_pools(lens, prefixes, page, KVH, 16, case)
    q = torch.randn(sum(new), H, 16, generator=torch.Generator().manual_seed(case), dtype=torch.float64)
    want = _formula(q, k, v, table, lens, new)
    plan = PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new, prefixes=prefixes, device="cpu", fixed=fixed)
    # float64 sums of up to 5000 terms
    assert torch.allclose(_carry_out(q, k, v, table, plan), want, rtol=1e-10, atol=1e-12)
    assert torch.allclose(paged_attention(q, k, v, table, plan), want, rtol=1e-10, atol=1e-12)
    assert plan.positions.tolist() == [n - t + i for n, t in zip(lens, new) for i in range(t)]


def test_plan_update():
    """An update is the plan of the new lengths; a fixed plan's launches stay as
    they are, from the shortest to the longest lengths."""
    lens, new = [200, 300, 180], [1, 2, 1]
    shared = [([0, 2], 128)]
    for fixed in (False, True):
        plan = PagedPlan(lens, heads=4, kv_heads=2, new_tokens=new, prefixes=shared, device="cpu", fixed=fixed)
        held = plan._data
        size = lambda i: (i.tokens, i.groups, i.items, i.merge_tokens, i.records, i.ints)  # noqa: E731
        first = size(plan._info)
        for other in ([129, 2, 140], [4000, 9000, 129], [200, 300, 180]):
            plan.update(other)
            k, v, table = _shared_pools(other, shared, 8, 2, 16, 5)
            q = torch.randn(4, 4, 16, generator=torch.Generator().manual_seed(6), dtype=torch.float64)
            assert torch.allclose(_carry_out(q, k, v, table, plan), _formula(q, k, v, table, other, new), rtol=1e-10,
                                  atol=1e-12)
            assert plan.seq_lens == other
            assert not fixed or (size(plan._info) == first and plan._data is held)
    with pytest.raises(RuntimeError, match="128 tokens are not common to sequence 2"):
        plan.update([200, 300, 128])
    with pytest.raises(ValueError):
        plan.update([200, 300])
    assert plan.seq_lens == [200, 300, 180]


def test_plan_refusals():
    ok = dict(heads=4, kv_heads=2, device="cpu")
    for lens, kw, text in [([-1], {}, "0 or more"), ([4], {"new_tokens": [-1]}, "0 or more"), ([4], {"heads": 5}, "divisible"),
                           ([4], {"kv_heads": 0}, "divisible"), ([4], {"rows": [-2]}, "row -2"),
                           ([9, 9], {"prefixes": [([0, 1], 9)]}, "are not common"),
                           ([9, 9], {"prefixes": [([0, 1], -1)]}, "are not common"),
                           ([4], {"heads": 257, "kv_heads": 1}, "up to 256 query heads"),
                           ([4], {"new_tokens": [1 << 30]}, "too many new tokens")]:
        with pytest.raises(RuntimeError, match=text):
            PagedPlan(lens, **{**ok, **kw})
    for lens, kw in [([4], {"new_tokens": [1, 1]}), ([4], {"rows": []}), ([4, 4], {"prefixes": [([0, 2], 1)]}),
                     ([4, 4], {"prefixes": [([0], 1), ([1, 0], 1)]}), (4, {}), ([1 << 31], {})]:
        with pytest.raises(ValueError):
            PagedPlan(lens, **{**ok, **kw})


def test_shared_prefixes_found():
    """The groups that a cache finds: by pages, whole ones before the new
    tokens, the length that saves the most reading."""
    cache = _cache(pages=400, page=8, seqs=20, max_len=400)
    a, other = cache.add([100, 50])
    kids = cache.fork(a, 3)
    cache.extend([a, *kids], [1, 2, 3, 100])
    deep = cache.fork(kids[2], 2)
    cache.extend([kids[2], *deep], 1)
    seqs = [other, kids[0], a, deep[1], kids[1], kids[2], deep[0]]
    plan = cache.plan(seqs, heads=2)
    assert plan.rows == seqs and plan.seq_lens == cache.lengths(seqs)
    # 12 whole pages for all six: saves 60 page reads; 24 (of 200 tokens, 25 with the copied ones) for three: 48
    assert plan.prefixes == [([1, 2, 3, 4, 5, 6], 96)]
    assert cache.plan([a, kids[0]], heads=2).prefixes == [([0, 1], 96)]
    assert cache.plan([deep[0], a, deep[1]], heads=2).prefixes == [([0, 2], 200)]
    assert cache.plan([a, other], heads=2).prefixes == []
    # new tokens are never shared, nor pages that they begin in
    assert cache.plan([a, kids[0]], heads=2, new_tokens=[30, 1]).prefixes == [([0, 1], 64)]
    b, = cache.add([64])
    assert cache.plan([b, *cache.fork(b, 1)], heads=2).prefixes == [([0, 1], 56)]
    e = cache.add([0, 0])
    assert cache.plan(e, heads=2, new_tokens=0).prefixes == []


def test_plan_refuses_negative_new_tokens():
    """Refused before a page is looked up behind a sequence's end."""
    cache = _cache()
    empty, (a,) = cache.add([0, 0]), cache.add([40])
    forks = [a, *cache.fork(a, 3)]
    for seqs, new in ((empty, -16), (forks, -1), (forks, [1, 1, 1, -1000000000]), (forks, -(1 << 31))):
        with pytest.raises(RuntimeError, match="0 or more new tokens"):
            cache.plan(seqs, 1, new_tokens=new)
    assert cache.plan(forks, 1, new_tokens=1000).prefixes == []


# ------------------------------------------------------------ expressions
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_expressions(dtype):
    lens, new, prefixes = [70, 9, 130, 0, 2], [3, 9, 1, 2, 4], []
    k, v, table = _shared_pools(lens, prefixes, 8, 2, 32, 3, dtype=dtype)
    q = torch.randn(sum(new), 6, 32, generator=torch.Generator().manual_seed(3)).to(dtype)
    plan = PagedPlan(lens, heads=6, kv_heads=2, new_tokens=new, device="cpu")
    eps = torch.finfo(dtype).eps / 2
    for scale in (None, 0.3):
        out = paged_attention(q, k, v, table, plan, scale=scale)
        want = _formula(q, k, v, table, lens, new, scale)
        # the output's rounding, and float32 throughout: scores below 32 over 32 products, relative to each probability
        bound = eps * want.abs() + (0 if dtype == torch.float64 else 1) * 64 * 32 * 2.0 ** -24 * 5 + 1e-12
        assert out.dtype == dtype and ((out.double() - want).abs() <= bound).all()
    single = paged_attention(q[:2], k, v, table, [70, 9])
    assert torch.equal(single, paged_attention(q[:2], k, v, table, PagedPlan([70, 9], heads=6, kv_heads=2, device="cpu")))


def test_expressions_differentiate():
    lens, new = [12, 3, 1], [2, 3, 2]
    k, v, table = _shared_pools(lens, [], 8, 1, 16, 4)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    q = torch.randn(7, 2, 16, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    plan = PagedPlan(lens, heads=2, kv_heads=1, new_tokens=new, device="cpu")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    assert torch.autograd.gradcheck(lambda *a: paged_attention(*a, table, plan), leaves)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_rope_append_expressions(dtype):
    lens, new = [70, 9, 130, 0, 2], [3, 9, 1, 2, 4]
    k, v, table = _shared_pools(lens, [], 8, 2, 32, 5, dtype=dtype)
    plan = PagedPlan(lens, heads=4, kv_heads=2, new_tokens=new, device="cpu")
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn(plan.tokens, 8, 32, generator=g).to(dtype)
    cos, sin = (torch.randn(plan.tokens, 32, generator=g).to(dtype) for _ in range(2))
    k0, v0 = k.clone(), v.clone()
    q = rope_append(qkv, cos, sin, k, v, table, plan)
    x = qkv.double()
    want = x * cos.double()[:, None] + torch.cat([-x[..., 16:], x[..., :16]], -1) * sin.double()[:, None]
    size = x.abs() * cos.double().abs()[:, None] + x.abs().roll(16, -1) * sin.double().abs()[:, None]
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 3 * 2.0 ** -24 * size  # and two products and a sum in float32
    assert ((q.double() - want[:, :4]).abs() <= bound[:, :4]).all()
    t = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for i in range(m):
            pos = n - m + i
            if pos >= 0:
                p, r = int(table[b, pos // 8]), pos % 8
                assert ((k[p, r].double() - want[t, 4:6]).abs() <= bound[t, 4:6]).all()
                assert torch.equal(v[p, r], qkv[t, 6:])
                k[p, r], v[p, r] = k0[p, r], v0[p, r]
            t += 1
    assert torch.equal(k.nan_to_num(9.0), k0.nan_to_num(9.0)) and torch.equal(v.nan_to_num(9.0), v0.nan_to_num(9.0))


def test_later_values_stay_out():
    """Infinities and NaN of tokens that a row does not attend to leave it as it
    is; those that it attends to are in their own dims."""
    g = torch.Generator().manual_seed(0)
    lens, new = [20, 9, 2], [6, 9, 4]
    k, v, table = _shared_pools(lens, [], 8, 2, 16, 1)
    q = torch.randn(sum(new), 4, 16, generator=g, dtype=torch.float64)
    plan = PagedPlan(lens, heads=4, kv_heads=2, new_tokens=new, device="cpu")
    clean = paged_attention(q, k, v, table, plan)
    at = {0: (17, 3, math.inf), 1: (4, 7, math.nan), 2: (1, 0, -math.inf)}
    for b, (n, d, x) in at.items():
        v[table[b, n // 8].long(), n % 8, 1, d] = x
    out = paged_attention(q, k, v, table, plan)
    t0 = 0
    for b, (n, d, x) in at.items():
        for i in range(new[b]):
            sees = lens[b] - new[b] + i >= n
            hit = torch.zeros(4, 16, dtype=torch.bool)
            hit[2:, d] = sees
            assert torch.equal(out[t0 + i][~hit], clean[t0 + i][~hit]), (b, i)
            want = torch.full((2,), x, dtype=torch.float64)
            assert not sees or torch.equal(out[t0 + i][hit].nan_to_num(9.0), want.nan_to_num(9.0)), (b, i)
        t0 += new[b]


def test_call_refusals():
    k, v, table = _shared_pools([20, 9], [], 8, 2, 16, 1)
    plan = PagedPlan([20, 9], heads=4, kv_heads=2, device="cpu")
    q = torch.zeros(2, 4, 16, dtype=torch.float64)
    qkv, cs = torch.zeros(2, 8, 16, dtype=torch.float64), torch.zeros(2, 16, dtype=torch.float64)
    short = PagedPlan([20, 70], heads=4, kv_heads=2, device="cpu")
    far = PagedPlan([20], heads=4, kv_heads=2, rows=[2], device="cpu", new_tokens=2)
    for call in [
        lambda: paged_attention(q[:1], k, v, table, plan), lambda: paged_attention(q[:, :2], k, v, table, plan),
        lambda: paged_attention(q[0], k, v, table, plan), lambda: paged_attention(q.float(), k, v, table, plan),
        lambda: paged_attention(q, k[:, :7], v[:, :7], table, plan), lambda: paged_attention(q, k, v[:-1], table, plan),
        lambda: paged_attention(q, k[:, :, :1], v[:, :, :1], table, plan),
        lambda: paged_attention(q, k[..., :8], v[..., :8], table, plan),
        lambda: paged_attention(q, k, v, table.long(), plan), lambda: paged_attention(q, k, v, table[0], plan),
        lambda: paged_attention(q, k, v, table.t().contiguous().t(), plan),
        lambda: paged_attention(q, k, v, table, short), lambda: paged_attention(q, k, v, table, far),
        lambda: paged_attention(q, k[:0], v[:0], table, plan),
        lambda: paged_attention(q, k, v, table, plan, scale=0.0), lambda: paged_attention(q, k, v, table, plan, scale=-1.0),
        lambda: paged_attention(q, k, v, table, plan, scale=float("inf")),
        lambda: paged_attention(q, k, v, table, plan, scale=float("nan")),
        lambda: rope_append(qkv[:1], cs, cs, k, v, table, plan), lambda: rope_append(qkv, cs[:1], cs, k, v, table, plan),
        lambda: rope_append(qkv, cs.float(), cs, k, v, table, plan), lambda: rope_append(qkv, cs, cs, k, v, table, short),
        lambda: rope_append(qkv.float(), cs.float(), cs.float(), k, v, table, plan),
    ]:
        with pytest.raises(ValueError):
            call()


def test_sizes_that_are_refused():
    """Lengths past the kernel's 32-bit positions, counts that do not fit, and
    numbers that would wrap: refused, with nothing changed."""
    for lens, kw in (([(1 << 30) + 1], {}), ([(1 << 31) - 1], {}), ([5], {"new_tokens": 1 << 30}),
                     ([5], {"new_tokens": (1 << 26) + 1}), ([5] * 70, {"new_tokens": 1 << 20})):
        with pytest.raises(RuntimeError):
            PagedPlan(lens, heads=1, kv_heads=1, device="cpu", **kw)
    assert PagedPlan([1 << 30], heads=1, kv_heads=1, device="cpu").tokens == 1
    for heads in ((1 << 32) + 4, 1 << 40):
        with pytest.raises(ValueError):
            PagedPlan([5], heads=heads, kv_heads=1, device="cpu")
    cache = _cache()
    a, = cache.add([5])
    for call in (lambda: cache.fork(a, 1 << 40), lambda: cache.fork(a, cache.max_seqs + 1), lambda: cache.fork(a, -1),
                 lambda: cache.pages((1 << 32) + a)):
        with pytest.raises(ValueError):
            call()
    assert cache.used_pages == 1 and cache.lengths([a]) == [5]


def test_inference_mode():
    """A cache and a plan made in inference mode are used outside of it."""
    with torch.inference_mode():
        cache = _cache()
        a, = cache.add([9])
        plan = cache.plan([a], 2)
    b, = cache.fork(a)
    cache.extend([b], 3)
    plan.update([8])
    q = torch.zeros(1, 2, 16)
    assert paged_attention(q, cache.k[0], cache.v[0], cache.block_table, plan).shape == q.shape


def test_library_refusals():
    """The C entries check what they are given before anything is launched."""
    lib = paged._lib()
    error = lambda: lib.santa_last_error().decode()  # noqa: E731
    plan = PagedPlan([20, 9], heads=4, kv_heads=2, device="cpu")
    info, one = ctypes.byref(plan._info), ctypes.c_void_p(16)
    strides = (ctypes.c_longlong * 8)(512, 128, 2048, 256, 128, 2048, 256, 128)

    def attend(q=one, dtype=0, D=128, pages=4, page=8, st=strides, width=4, rows=2, ws=one, size=1 << 30, scale=1.0):
        return lib.santa_paged_attention(q, one, one, one, dtype, D, pages, page, st, one, width, rows, info, one, scale,
                                         ws, size, None)

    odd = (ctypes.c_longlong * 8)(512, 128, 2048, 256, 4, 2048, 256, 128)
    for kw, text in [({"q": None}, "bad paged_attention"), ({"dtype": 3}, "bad paged_attention"), ({"D": 96}, "64 or 128"),
                     ({"pages": 0}, "num_pages"), ({"page": 12}, "power of two"), ({"st": odd}, "multiples of 8"),
                     ({"width": 2}, "too narrow"), ({"rows": 1}, "row 1 of 1"),
                     ({"scale": 0.0}, "positive"), ({"scale": -1.0}, "positive"), ({"scale": 3e38}, "positive"),
                     ({"scale": float("nan")}, "positive"), ({"q": ctypes.c_void_p(8)}, "16-byte")]:
        assert attend(**kw) != 0 and text in error(), (kw, error())
    if plan._info.records:
        assert attend(size=8) == 3 and attend(ws=None) == 1
    pools = (ctypes.c_void_p * 1)(16)
    for args, text in [((pools, 1, 24, 32, 4), "16-byte"), ((pools, 1, 32, 16, 4), "16-byte"),
                       (((ctypes.c_void_p * 1)(8), 1, 32, 32, 4), "aligned")]:
        assert lib.santa_paged_copy(*args, (ctypes.c_int * 2)(0, 1), 1, None) == 1 and text in error()
    for pairs, text in [((0, 4), "no page"), ((0, 1, 2, 1), "written twice"), ((0, 1, 1, 2), "both read")]:
        assert lib.santa_paged_copy(pools, 1, 32, 32, 4, (ctypes.c_int * len(pairs))(*pairs), len(pairs) // 2, None) == 1
        assert text in error()
    assert lib.santa_pages_add(None, None, 0, None) == 1 and lib.santa_pages_compact(None) == 1
    assert lib.santa_pages_length(None, 0) == -1 and lib.santa_pages_used(None) == -1
    small = (ctypes.c_int * 4)()
    out = paged._PlanInfo()
    made = lib.santa_paged_plan(small, small, None, 2, None, None, 0, 4, 2, 0, ctypes.byref(out), small, 1)
    assert made != 0 or out.ints <= 1


# -------------------------------------------------------------------- model
TINY = LlamaShape(hidden=128, intermediate=256, heads=8, kv_heads=2, layers=2, vocab=97)


def _model_cache(shape, device="cpu", dtype=torch.float32, **kw):
    args = dict(num_pages=60, page_size=8, max_seqs=8, max_len=120, kv_heads=shape.kv_heads, head_dim=shape.head_dim)
    return PagedKVCache(shape.layers, dtype=dtype, device=device, **{**args, **kw})


def test_model_extends():
    """Prompts, prompts behind a forked one and single tokens, after pages have
    moved: the logits are those of each sequence prefilled by itself."""
    model = RandomLlama(TINY, seed=3, std=0.05, dtype=torch.float32, device="cpu")
    g = torch.Generator().manual_seed(2)
    toks = torch.randint(0, TINY.vocab, (4, 100), generator=g)
    toks[1:, :30] = toks[0, :30]  # three sequences share 30 tokens with the first

    def alone(s, n):
        return model.prefill(toks[s:s + 1, :n], NHDCache(TINY, 1, n, torch.float32, "cpu"))[0]

    cache = _model_cache(TINY)
    gone, a = cache.add([40, 0])
    close = lambda x, y: (x - y).abs().max() < 1e-5  # noqa: E731
    assert close(model.extend(toks[:1, :30], cache, [a])[0], alone(0, 30))
    b, c = cache.fork(a, 2)
    logits = model.extend(torch.cat([toks[2, 30:49], toks[0, 30:31], toks[1, 30:37]]), cache, [c, a, b], [19, 1, 7],
                          mlp_chunk=5)
    assert all(close(x, alone(s, n)) for x, s, n in zip(logits, (2, 0, 1), (49, 31, 37)))
    d, = cache.fork(b)
    toks[3, :37] = toks[1, :37]
    cache.free([gone])
    cache.compact()
    lens = dict(zip((a, b, c, d), (31, 37, 49, 37)))
    for i in range(4):
        order = [d, a, c, b]
        backend = ExactDecodeBackend() if i == 2 else None
        logits = model.extend(torch.stack([toks[(a, b, c, d).index(s), lens[s]] for s in order]), cache, order, 1,
                              backend=backend)
        for s, x in zip(order, logits):
            lens[s] += 1
            assert close(x, alone((a, b, c, d).index(s), lens[s]))
    assert cache.lengths([a, b, c, d]) == [lens[s] for s in (a, b, c, d)]
    used = cache.used_pages
    for bad in (lambda: model.extend(toks[:2, :3], cache, [a]), lambda: model.extend(toks[0, :3], cache, [a, b], [3, 0]),
                lambda: model.extend(toks[0, :3], cache, [a, b], [1, 1]), lambda: model.extend(toks[0, :0], cache, [], []),
                lambda: model.extend(toks[:1, :3], cache, [a], backend=ExactDecodeBackend()),
                lambda: model.extend(toks[:1, :3], _model_cache(TINY, page_size=16, head_dim=32), [0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="would hold"):
        model.extend(toks[:1, :99], cache, [a])
    assert cache.used_pages == used


def test_model_refuses_before_the_cache_changes():
    """Tokens that the model has no embedding for leave the cache as it was."""
    model = RandomLlama(TINY, device="cpu", dtype=torch.float32, seed=1)
    cache = _model_cache(TINY)
    a, = cache.add([0])
    with pytest.raises(IndexError):
        model.extend(torch.full((1, 3), TINY.vocab), cache, [a])
    assert cache.lengths([a]) == [0] and cache.used_pages == 0


def test_backend_decodes_pages():
    lens = [20, 9, 64]
    k, v, table = _shared_pools(lens, [], 8, 2, 32, 3, dtype=torch.float32)
    q = torch.randn(3, 4, 32, generator=torch.Generator().manual_seed(1))
    want = paged_attention(q, k, v, table, lens)
    for x in (lens, torch.tensor(lens)):
        assert torch.equal(ExactDecodeBackend().decode_paged(q, k, v, table, x), want)
    same = ExactDecodeBackend().decode_paged(q, k, v, table, 9)
    assert torch.equal(same, paged_attention(q, k, v, table, [9, 9, 9]))


def test_backend_decodes_a_plan(monkeypatch):
    """One plan for all layers, with prefixes and rows of a whole block table;
    RandomLlama.extend hands its own over."""
    lens, shared = [70, 66, 90], [([0, 2], 64)]
    k, v, table = _shared_pools(lens, shared, 8, 2, 32, 3, dtype=torch.float32)
    q = torch.randn(3, 4, 32, generator=torch.Generator().manual_seed(1))
    wide = torch.full((6, table.shape[1]), 1 << 30, dtype=torch.int32)
    wide[[4, 1, 5]] = table
    plan = PagedPlan(lens, heads=4, kv_heads=2, prefixes=shared, rows=[4, 1, 5], device="cpu")
    want = ExactDecodeBackend().decode_paged(q, k, v, table, lens)
    assert torch.equal(ExactDecodeBackend().decode_paged(q, k, v, wide, plan), want)
    with pytest.raises(ValueError, match="the plan is for 3 tokens"):
        ExactDecodeBackend().decode_paged(q[:2], k, v, wide, plan)
    model, cache = RandomLlama(TINY, seed=3, std=0.05, dtype=torch.float32, device="cpu"), _model_cache(TINY)
    a, = cache.add([0])
    model.extend(torch.arange(40)[None], cache, [a])
    made, given = [], []
    build, decode = PagedPlan.update, ExactDecodeBackend.decode_paged
    monkeypatch.setattr(PagedPlan, "update", lambda self, *args: made.append(self) or build(self, *args))
    monkeypatch.setattr(ExactDecodeBackend, "decode_paged", lambda self, *args: given.append(args[4]) or decode(self, *args))
    model.extend(torch.tensor([5, 6]), cache, [a, *cache.fork(a)], 1, backend=ExactDecodeBackend())
    assert len(made) == 1 and given == made * TINY.layers and made[0].prefixes == [([0, 1], 40)]


def test_model_refuses_chunks_without_tokens():
    """A negative chunk would leave the layers' MLPs out."""
    model, cache = RandomLlama(TINY, device="cpu", dtype=torch.float32, seed=1), _model_cache(TINY)
    a, = cache.add([0])
    for chunk in (0, -5):
        with pytest.raises(ValueError, match="mlp_chunk"):
            model.extend(torch.zeros(1, 3, dtype=torch.long), cache, [a], mlp_chunk=chunk)
    assert cache.lengths([a]) == [0]


def test_shrink():
    """Tokens leave from the end; pages that are left without any are given up,
    shared ones by one holder; refused for more than there are."""
    cache = _cache()
    a, b = cache.add([20, 9])
    lib, ints = paged._lib(), lambda *x: (ctypes.c_int * len(x))(*x)
    c, = cache.fork(a)
    cache.extend([c], 10)  # copies the last page
    pages, used = cache.pages(c), cache.used_pages
    cache._take_back([c, b], [10, 0])
    assert cache.lengths([a, b, c]) == [20, 9, 20] and cache.pages(c) == pages[:3] and cache.used_pages == used - 1
    cache._take_back([c], [13])
    assert cache.pages(c) == pages[:1] == cache.pages(a)[:1] and cache.used_pages == used - 2
    for seqs, tokens, text in (([c], [8], "8 tokens cannot leave"), ([a, b], [1, -1], "-1 tokens cannot leave"),
                               ([a, a], [1, 1], "named twice"), ([5], [1], "no sequence 5")):
        with pytest.raises(RuntimeError, match=text):
            cache._take_back(seqs, tokens)
    assert lib.santa_pages_shrink(None, ints(0), ints(0), 1) != 0
    assert lib.santa_pages_shrink(cache._pages, ints(0), None, 1) != 0
    cache._take_back([a, b, c], [20, 9, 7])
    assert cache.lengths([a, b, c]) == [0, 0, 0] and cache.used_pages == 0 and cache.compact() == 0


def test_model_takes_tokens_back():
    """A call that fails behind the lengthening leaves every sequence with the
    tokens that it had, and the next one goes on from there."""
    model, cache = RandomLlama(TINY, device="cpu", dtype=torch.float32, seed=1), _model_cache(TINY)
    a, = cache.add([0])
    first = torch.arange(19)[None]
    model.extend(first, cache, [a])
    seqs = [a, *cache.fork(a)]

    class Refuses:
        def decode_paged(self, *args):
            raise RuntimeError("This build supports only D=128")

    for backend in (Refuses(), object()):
        with pytest.raises((RuntimeError, AttributeError)):
            model.extend(torch.tensor([3, 4]), cache, seqs, 1, backend=backend)
        assert cache.lengths(seqs) == [19, 19]
    two = RandomLlama(TINY, device="cpu", dtype=torch.float32, seed=1)
    two.layers[1]["wo"] = two.layers[1]["wo"][:, :-1]
    with pytest.raises(RuntimeError):
        two.extend(torch.arange(40)[None], cache, seqs, [30, 10])
    assert cache.lengths(seqs) == [19, 19] and cache.used_pages == 4  # the copied last page stays one
    logits = model.extend(torch.tensor([3, 4]), cache, seqs, 1)
    for t, x in zip((3, 4), logits):
        want = model.prefill(torch.cat([first, torch.tensor([[t]])], 1), NHDCache(TINY, 1, 20, torch.float32, "cpu"))[0]
        assert (x - want).abs().max() < 1e-5


def test_captured_plans_are_held():
    """What a captured call has room for bounds later updates; where a replay
    would not follow an update, there is none."""
    args = dict(heads=2, kv_heads=1, device="cpu")
    plan = PagedPlan([20, 30], fixed=True, **args)
    plan._captured(10, True)  # nothing is captured here
    plan._hold(100)
    plan._hold(80)
    plan.update([80, 1])
    with pytest.raises(RuntimeError, match="81 > 80"):
        plan.update([5, 81])
    assert plan.seq_lens == [80, 1]
    plan._hold(-1)
    loose = PagedPlan([20, 30], **args)
    loose._hold(-1)
    for p in (plan, loose):
        with pytest.raises(RuntimeError, match="a captured call holds"):
            p.update([5, 5])


def test_plans_are_built_once(monkeypatch):
    """The buffer is large enough at first, of whatever shape the batch is; one
    that is not is made again."""
    lib, calls = paged._lib(), []

    class Counted:
        def __getattr__(self, name):
            if name == "santa_paged_plan":
                return lambda *args: calls.append(args[-1]) or lib.santa_paged_plan(*args)
            return getattr(lib, name)

    monkeypatch.setattr(paged, "_lib_ready", Counted())
    r = random.Random(1)
    for _ in range(60):
        KVH, GH, B = r.choice((1, 2, 8, 32)), r.choice((1, 4, 7, 16, 40, 128, 255)), r.randint(0, 40)
        new = [r.choice((0, 1, 1, 5, 300)) for _ in range(B)]
        lens = [r.choice((0, 1, 100, 5000, 70000)) + 400 for _ in range(B)]
        order = r.sample(range(B), B)
        cut = r.randint(0, B)
        calls.clear()
        plan = PagedPlan(lens, heads=KVH * GH, kv_heads=KVH, new_tokens=new, device="cpu", fixed=r.random() < 0.5,
                         prefixes=[(order[:cut], 70), (order[cut:], 64)])
        plan.update(lens)
        assert len(calls) == 2 and len(plan._data) == max(1, plan._info.ints)
    calls.clear()
    plan = PagedPlan([5, 70], heads=2, kv_heads=2, device="cpu")
    want = plan._data.clone()
    plan._size = 3
    plan.update([5, 70])
    assert calls[1:] == [3, len(want)] and torch.equal(plan._data, want)
    with pytest.raises(RuntimeError, match="0 or more"):
        plan.update([5, -1])


def test_page_lists_grow_in_steps():
    """A sequence that gains its pages one by one does not move its list each time."""
    cache = _cache(pages=1000, page=8, seqs=1, max_len=8000, layers=0)
    a, = cache.add([0])
    row, seen = ctypes.POINTER(ctypes.c_int)(), []
    for i in range(1000):
        cache.extend([a], 8)
        assert paged._lib().santa_pages_row(cache._pages, a, ctypes.byref(row)) == i + 1
        seen.append(ctypes.addressof(row.contents))
    assert sum(x != y for x, y in zip(seen, seen[1:])) <= 10 and cache.pages(a) == list(range(1000))


def test_numbers_that_are_not_whole():
    """2.5 tokens are none: refused, where they were cut off; any kind of whole
    numbers is taken, iterators among them."""
    cache = _cache()
    a, b = cache.add(x for x in (3.0, 5))
    for call in (lambda: cache.add([2.5]), lambda: cache.extend([a], [0.5]), lambda: cache.free([a + 0.5]),
                 lambda: cache.plan([a], 1, [0.5]), lambda: PagedPlan([4.5], heads=1, kv_heads=1, device="cpu"),
                 lambda: PagedPlan(torch.tensor([4.5]), heads=1, kv_heads=1, device="cpu"),
                 lambda: copy_pages(cache.k, [0.5], [1]), lambda: cache.lengths([float("nan")])):
        with pytest.raises(ValueError):
            call()
    assert cache.lengths(iter([b, a])) == [5, 3] and cache.lengths(torch.tensor([a, b]).numpy()) == [3, 5]
    with pytest.raises(RuntimeError, match="no sequence 7"):
        cache.lengths(x for x in (a, 7))


def test_which_plans_round():
    """Several new tokens with more than 32 rows in a sequence; never single ones."""
    for new, GH, want in (([1, 1], 256, 0), ([1, 0], 33, 0), ([8, 1], 4, 0), ([1, 9], 4, 1), ([2], 16, 0), ([2], 17, 1),
                          ([0], 4, 0), ([300], 1, 1)):
        plan = PagedPlan([400] * len(new), heads=2 * GH, kv_heads=2, new_tokens=new, device="cpu")
        assert plan._info.rounded == want, (new, GH)
