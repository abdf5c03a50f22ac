"""The tile pipeline of the attention over pages in its steady state: items of
many tiles, so that the ring of tiles wraps, every wait is met and pages are
looked up anew, in every form that a wave's work has, and workgroups that go from
one form to another.  64 KV heads leave four workgroups for each, so the items
are long; what a case is meant to reach is checked on its plan.

Every case prints its name before touching the GPU.
"""
import math

import pytest
import torch

from santa_amd.paged import PagedPlan, paged_attention
from test_shared_pages_gpu import _check

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
KVH, GH = 64, 4


def _chains(plan):
    """Of every workgroup, (rows, tiles) of its items one after the other."""
    info = plan._info
    items = plan._data[:16 * info.items].view(-1, 16)[:, :9].cpu().tolist()
    out = []
    for w in range(info.groups):
        out.append([])
        while w >= 0 and items[w][5] > 0:
            _, _, begin, end, _, rows, _, _, w = items[w]
            out[-1].append((rows, -(-(end - begin) // 64)))
    return out


def _form(rows):
    return sum(rows > n for n in (16, 32, 64, 128))


def _pools(lens, shared, page, D, dtype, seed):
    """Pools in random page order; the first `shared` tokens of all sequences in
    the same pages; NaN wherever no token is."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    common, used = shared // page, [-(-n // page) for n in lens]
    total = common + sum(u - common for u in used) + 2
    k, v = (torch.randn(total, page, KVH, D, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(lens), max(used) + 3), int(order[0]), dtype=torch.int32)
    k[order[:2].cuda()], v[order[:2].cuda()] = math.nan, math.nan
    at = 2 + common
    for b, u in enumerate(used):
        table[b, :common] = order[2:2 + common].int()
        table[b, common:u] = order[at:at + u - common].int()
        at += u - common
        if lens[b] % page:
            for t in (k, v):
                t[int(table[b, u - 1]), lens[b] % page:] = math.nan
    return k, v, table.cuda()


def _formula(q, k, v, table, lens, new):
    """test_shared_pages_gpu._reference, all query heads of a KV head at once."""
    N, H, D = q.shape
    page, scale = k.shape[1], 1.0 / math.sqrt(D)
    out, mean, off = (torch.zeros(N, H, D, dtype=torch.float64, device="cuda") for _ in range(3))
    t0 = 0
    for b, (n, t) in enumerate(zip(lens, new)):
        at = torch.arange(n, device="cuda")
        ks, vs = (x[table[b, at // page].long(), at % page] for x in (k, v))
        pos = torch.arange(n - t, n, device="cuda").repeat_interleave(GH)
        later = at[None, :] > pos[:, None]
        for h in range(KVH):
            kh, vh = ks[:, h].double(), vs[:, h].double()
            x = q[t0:t0 + t, h * GH:(h + 1) * GH].double().reshape(-1, D)
            p = torch.softmax((x @ kh.t().contiguous() * scale).masked_fill(later, -math.inf), -1)
            size = (x.abs() @ kh.t().abs().contiguous() * scale).masked_fill(later, 0.0).amax(-1)
            bound = (2 * (D + 2) * 2.0 ** -24 * size + 2.0 ** -20)[:, None].expand(-1, D)
            for to, y in ((out, p @ vh), (mean, p @ vh.abs()), (off, bound)):
                to[t0:t0 + t, h * GH:(h + 1) * GH] = y.reshape(t, GH, D)
        t0 += t
    return out, mean, off


def _run(lens, new, shared, page, D, dtype, seed):
    k, v, table = _pools(lens, shared, page, D, dtype, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(sum(new), KVH * GH, D, generator=g, device="cuda").mul(1.5).to(dtype)
    prefixes = [(list(range(len(lens))), shared)] if shared else []
    plan = PagedPlan(lens, heads=KVH * GH, kv_heads=KVH, new_tokens=new, prefixes=prefixes)
    want = _formula(q, k, v, table, lens, new)
    for rounded in (False, True):
        _check(paged_attention(q, k, v, table, plan, rounded=rounded), want, dtype)
    return plan


# new tokens a sequence: 4, 28, 60, 124 and 256 rows
FORMS = [1, 7, 15, 31, 64]


@pytest.mark.parametrize("D, dtype, page", [(128, BF, 16), (64, F16, 8), (64, BF, 64), (128, F16, 256)])
@pytest.mark.parametrize("tokens", FORMS)
def test_long_items(tokens, D, dtype, page):
    """Every workgroup holds more than 128 tiles of one form, odd numbers of tiles
    among them, ends inside a tile, a page and eight tokens."""
    lens = [8257, 8386, 8500, 8321, 8192 + 64 * 3]
    print(f"\n[case] long items tokens={tokens} D={D} {dtype} page={page}", flush=True)
    new = [tokens] * len(lens)
    chains = _chains(_run(lens, new, 0, page, D, dtype, tokens + D))
    items = [i for c in chains for i in c]
    assert {_form(rows) for rows, _ in items} == {_form(4 * tokens)} and len(chains) == 4
    assert max(tiles for _, tiles in items) > 128 and any(tiles > 64 and tiles % 2 for _, tiles in items)


@pytest.mark.parametrize("D, dtype, page, shared", [(128, BF, 16, 0), (64, F16, 32, 0), (128, F16, 64, 4480), (64, BF, 8, 4416)])
def test_changing_forms(D, dtype, page, shared):
    """Workgroups that go through items of several forms, with more and fewer
    tiles than the ring holds, whose loads run ahead from one into the next."""
    lens = [8300, 4700, 6500, 5000, 7777, 4600, 4545, 4500, 9001, 4609, 4666]
    new = [1, 7, 15, 31, 64, 1, 7, 15, 2, 31, 70]
    if not shared:
        lens[5:8], lens[9:] = [130, 700, 64], [65, 90]
    print(f"\n[case] changing forms D={D} {dtype} page={page} shared={shared}", flush=True)
    chains = _chains(_run(lens, new, shared, page, D, dtype, D + shared))
    assert max(tiles for c in chains for _, tiles in c) > 64
    assert {_form(rows) for c in chains for rows, _ in c} == {0, 1, 2, 3, 4}
    assert max(len({_form(rows) for rows, _ in c}) for c in chains) >= 4
    steps = [(a, b) for c in chains for a, b in zip(c, c[1:])]
    assert any(a[1] > 8 and b[1] > 8 for a, b in steps) and (shared or any(a[1] < 3 for a, _ in steps))
