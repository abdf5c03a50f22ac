"""Shared paged caches on the GPU: the attention over pages, RoPE with the page
write, page copies and the block table, against float64 formulas and the CPU.

Tolerance of the attention: the output is rounded once (eps of its value, eps
= 2^-8 in bf16 and 2^-11 in f16); the probabilities are rounded once more where
more than 16 rows pass over a KV head's tokens together (eps of the mean of |v|
under them), else twice as finely (eps^2); float32 scores are off by at most
(D + 2) x 2^-24 of the sum of the |products|, and that, twice (a score and the
maximum, a score and the mass), is what a probability is off by, with another
2^-20 for its exponential and the float32 sums' growth.

Every case prints its name before touching the GPU.
"""
import math
import random

import pytest
import torch

from santa_amd.paged import PagedKVCache, PagedPlan, copy_pages, paged_attention, rope_append
from santa_amd import attention_backends as ab
from santa_amd.runtime import ExactDecodeBackend, LlamaShape, NHDCache, RandomLlama
from test_paged import _model_cache, _shared_pools

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def _reference(q, k, v, table, lens, new, scale=None):
    """(values, mean of |v|, bound of the scores' rounding) in float64, sequence by sequence and head by head."""
    N, H, D = q.shape
    page, KVH = k.shape[1:3]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, mean, off = (torch.zeros(N, H, D, dtype=torch.float64, device=q.device) for _ in range(3))
    t0 = 0
    for b, (n, t) in enumerate(zip(lens, new)):
        blind = min(t, max(0, t - n))
        if t > blind:
            at = torch.arange(n, device=q.device)
            rows = (table[b, at // page].long(), at % page)
            later = at[None, :] > torch.arange(n - t + blind, n, device=q.device)[:, None]
            span = slice(t0 + blind, t0 + t)
            for h in range(H):
                kh, vh = (x[rows][:, h // (H // KVH)].double() for x in (k, v))
                x = q[span, h].double()
                p = torch.softmax((x @ kh.t().contiguous() * scale).masked_fill(later, -math.inf), -1)
                out[span, h], mean[span, h] = p @ vh, p @ vh.abs()
                size = (x.abs() @ kh.t().abs().contiguous() * abs(scale)).masked_fill(later, 0.0).amax(-1)
                off[span, h] = (2 * (D + 2) * 2.0 ** -24 * size + 2.0 ** -20)[:, None]
        t0 += t
    return out, mean, off


def _check(out, ref, dtype, rounded=True):
    want, mean, off = ref
    eps = torch.finfo(dtype).eps / 2
    bound = eps * want.abs() + ((eps if rounded else eps * eps) + off) * (1 + eps) * mean
    if dtype == F16:
        bound += 2.0 ** -24  # the smallest f16 numbers: half a step of the output, and of a probability's second part
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all() and (err <= bound).all(), (err / bound.clamp_min(1e-30)).max().item()


def _case(lens, new, prefixes, H, KVH, D, page, dtype, seed=0, **kw):
    k, v, table = (t.cuda() for t in _shared_pools(lens, prefixes, page, KVH, D, seed, dtype=dtype))
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(sum(new), H, D, generator=g).mul(1.5).to("cuda", dtype)
    plan = PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new, prefixes=prefixes, **kw)
    return q, k, v, table, plan


# lengths around the tiles of 64, pages that end inside one, empty and short
# sequences; every head count from few rows to several blocks of them
CASES = [
    ([1], [1], [], 8, 2, 128, 16, BF), ([64], [1], [], 4, 4, 64, 8, F16),
    ([63, 65, 129], [1, 1, 1], [], 2, 1, 128, 8, BF),
    ([0, 7, 0, 200], [1, 1, 1, 1], [], 6, 2, 128, 32, F16), ([700], [1], [], 7, 1, 64, 64, BF),
    ([1000, 33], [1, 1], [], 32, 8, 128, 256, BF), ([500, 20], [1, 1], [], 17, 1, 128, 16, BF),
    ([500, 400], [1, 1], [], 40, 1, 64, 16, F16), ([300], [1], [], 128, 1, 128, 16, BF),
    ([300], [1], [], 33, 1, 128, 8, F16),
    # prefixes: all, some, two groups in any order, shorter than a tile, of a length inside a page and a tile
    ([200, 150, 131], [1, 1, 1], [([0, 1, 2], 128)], 8, 2, 128, 16, BF),
    ([400, 390, 380, 10], [1, 1, 1, 1], [([2, 0], 320)], 4, 1, 64, 32, F16),
    ([300, 200, 310, 250, 99], [1, 1, 1, 1, 1], [([3, 0], 200), ([1, 4, 2], 96)], 28, 4, 128, 8, BF),
    ([90, 80], [1, 1], [([0, 1], 56)], 8, 8, 128, 8, BF),
    ([2000] * 40, [1] * 40, [(list(range(40)), 1984)], 32, 8, 128, 16, BF),
    ([513 + i for i in range(70)], [1] * 70, [(list(range(70)), 512)], 8, 4, 64, 64, F16),
    # several new tokens, among them more than there are positions, and none
    ([300, 20, 2, 0], [5, 20, 7, 3], [], 4, 2, 128, 8, BF), ([130, 64], [130, 64], [], 8, 2, 64, 16, F16),
    ([700, 650, 300, 66], [90, 1, 0, 2], [([0, 1, 2, 3], 64)], 7, 1, 128, 32, BF),
    ([900, 850], [260, 300], [([0, 1], 512)], 32, 8, 128, 16, BF), ([1025], [1000], [], 12, 1, 64, 128, F16),
    ([200] * 5, [4] * 5, [(list(range(5)), 128)], 4, 1, 128, 64, F16), ([333], [40], [], 128, 2, 64, 8, BF),
]


@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_paged_attention(case, fixed):
    lens, new, prefixes, H, KVH, D, page, dtype = CASES[case]
    print(f"\n[case] paged attention {case} lens={lens[:6]} new={new[:6]} H={H} KVH={KVH} D={D} page={page} {dtype}",
          flush=True)
    q, k, v, table, plan = _case(lens, new, prefixes, H, KVH, D, page, dtype, case, fixed=fixed)
    out = paged_attention(q, k, v, table, plan)
    few = max(new) * H // KVH <= 16 and sum(new) * H // KVH <= 16
    _check(out, _reference(q, k, v, table, lens, new), dtype, rounded=not few)
    t0 = 0
    for n, t in zip(lens, new):
        assert (out[t0:t0 + max(0, t - n)] == 0).all()
        t0 += t
    assert torch.equal(out, paged_attention(q, k, v, table, plan))  # the same bits each time


def test_scale_and_lengths():
    print("\n[case] a scale of one's own; lengths in place of a plan", flush=True)
    lens = [300, 64, 5]
    q, k, v, table, plan = _case(lens, [1] * 3, [], 8, 2, 128, 16, BF)
    out = paged_attention(q, k, v, table, plan, scale=0.02)
    _check(out, _reference(q, k, v, table, lens, [1] * 3, 0.02), BF, rounded=False)
    assert torch.equal(paged_attention(q, k, v, table, lens), paged_attention(q, k, v, table, plan))
    assert torch.equal(paged_attention(q, k, v, table, torch.tensor(lens)), paged_attention(q, k, v, table, plan))


def test_large_scores():
    """Scores that grow with the position by far more than the 16-bit types
    resolve, and scores of 1e12 to 1e16: each row attends to its best token."""
    print("\n[case] growing and huge scores", flush=True)
    n, page = 500, 16
    for top in (8.0, 2.0 ** 20):
        q, k, v, table, _ = _case([n, n - 1], [1, 3], [], 24, 1, 128, page, BF)
        level = torch.randperm(n, generator=torch.Generator().manual_seed(3)).float() if top > 8 else torch.arange(n)
        rows = (table[:, torch.arange(n, device="cuda") // page].long(), torch.arange(n, device="cuda") % page)
        kk = (level.cuda() + 1).bfloat16() * top
        k[rows[0][0], rows[1], 0] = kk[:, None].expand(-1, 128)
        k[rows[0][1, :n - 1], rows[1][:n - 1], 0] = kk[:n - 1, None].expand(-1, 128)
        q = torch.full_like(q, top)
        plan = PagedPlan([n, n - 1], heads=24, kv_heads=1, new_tokens=[1, 3])
        out = paged_attention(q, k, v, table, plan)
        at = 0
        for b, m in ((0, n), (1, n - 3), (1, n - 2), (1, n - 1)):
            best = (kk[:m] == kk[:m].max()).nonzero()[:, 0]
            want = v[table[b, best // page].long(), best % page, 0].double().mean(0)
            # equal scores only: probabilities of exactly 1
            assert ((out[at].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20).all()
            at += 1


def test_infinite_scores_and_values():
    """Keys of -inf weigh nothing, whole parts of them included; a row with no
    other key is NaN, as torch's softmax gives; infinite values stay in their
    own dims and rows."""
    print("\n[case] infinite keys and values", flush=True)
    lens, page = [400, 330, 70], 8
    q, k, v, table, plan = _case(lens, [1, 1, 1], [([0, 1], 256)], 4, 1, 128, page, BF)
    q[..., 5] = 1.0
    rows = lambda b, lo, hi: (table[b, torch.arange(lo, hi, device="cuda") // page].long(),  # noqa: E731
                              torch.arange(lo, hi, device="cuda") % page)
    for b, hi in ((0, 300), (2, 70)):
        k[(*rows(b, 0, hi), 0, 5)] = -math.inf
    out = paged_attention(q, k, v, table, plan)
    assert out[2].isnan().all()
    want = _reference(q[:2], k, v, table, lens[:2], [1, 1])
    off = torch.where(want[2].isfinite(), want[2], 128 * 2.0 ** -17)  # the masked scores' own bound is not finite
    _check(out[:2], (want[0], want[1], off), BF, rounded=False)
    v[(*rows(0, 399, 400), 0, 7)] = math.inf
    out = paged_attention(q, k, v, table, plan)
    assert torch.equal(out.isinf(), torch.zeros_like(out, dtype=torch.bool).index_put_(
        (torch.zeros(4, dtype=torch.long, device="cuda"), torch.arange(4, device="cuda"),
         torch.full((4,), 7, device="cuda")), torch.ones(4, dtype=torch.bool, device="cuda")))
    assert out[:2].isfinite().sum() == 2 * 4 * 128 - 4


@pytest.mark.parametrize("lens, new, H, KVH, D, dtype", [
    ([70], [3], 4, 1, 128, BF), ([40, 129], [6, 7], 4, 1, 64, F16), ([130], [30], 2, 1, 128, F16),
    ([100, 3], [50, 5], 4, 2, 64, BF), ([300], [64], 4, 1, 128, BF), ([200], [150], 1, 1, 64, F16)])
def test_values_of_later_tokens_stay_out(lens, new, H, KVH, D, dtype):
    """Infinities and NaN among the values of a token that a row does not attend
    to leave the row as it is, bit for bit."""
    print(f"\n[case] values of later tokens lens={lens} new={new} H={H} D={D} {dtype}", flush=True)
    q, k, v, table, plan = _case(lens, new, [], H, KVH, D, 8, dtype)
    clean = paged_attention(q, k, v, table, plan)
    t0 = 0
    marks = []
    for b, (n, t) in enumerate(zip(lens, new)):
        for i, x in ((t - 1, math.nan), (t // 2, math.inf), (max(1, t - n + 1), -math.inf)):
            d = (7 * i + 5) % D
            v[table[b, (n - t + i) // 8].long(), (n - t + i) % 8, KVH - 1, d] = x
            marks.append((t0, t, i, d, x))
        t0 += t
    out = paged_attention(q, k, v, table, plan)
    hit = torch.zeros(out.shape, dtype=torch.bool)
    for at, t, i, d, _ in marks:
        hit[at + i:at + t, H - H // KVH:, d] = True
    assert torch.equal(out.cpu()[~hit], clean.cpu()[~hit])
    assert not out.cpu()[hit].isfinite().any()


def test_strides_and_views():
    """Pools interleaved in one tensor, head-major pages, a table that is part of a
    wider one or one row for all, q of a fused projection, odd addresses."""
    print("\n[case] strides", flush=True)
    lens, new = [300, 90, 64], [2, 1, 3]
    q, k, v, table, plan = _case(lens, new, [], 8, 2, 64, 16, F16, 7)
    want = paged_attention(q, k, v, table, plan)
    both = torch.stack([k, v], dim=1)
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    wide = torch.full((5, table.shape[1] + 9), 1 << 30, dtype=torch.int32, device="cuda")
    wide[1:4, 3:3 + table.shape[1]] = table
    part = wide[1:4, 3:3 + table.shape[1]]
    fused = torch.randn(6, 12, 64, device="cuda", dtype=F16)
    fused[:, :8] = q
    odd = torch.empty(q.numel() + 1, device="cuda", dtype=F16)[1:].view(q.shape).copy_(q)
    for args in [(q, both[:, 0], both[:, 1], table), (q, *heads, part), (fused[:, :8], k, v, part), (odd, k, v, table),
                 (q.transpose(1, 2).contiguous().transpose(1, 2), k, v, table)]:
        assert torch.equal(paged_attention(*args, plan), want)
    rows = PagedPlan(lens[::-1], heads=8, kv_heads=2, new_tokens=new[::-1], rows=[3, 2, 1])
    back = torch.cat([q[3:], q[2:3], q[:2]])
    got = paged_attention(back, k, v, wide[:, 3:3 + table.shape[1]], rows)
    assert torch.equal(torch.cat([got[4:], got[3:4], got[:3]]), want)
    one = paged_attention(q[:3], k, v, table[:1].expand(3, -1), [300, 200, 8])
    assert torch.equal(one[0], paged_attention(q[:1], k, v, table[:1], [300])[0])
    solo = k[:1].transpose(0, 3).contiguous().transpose(0, 3)[:, :8, :1]  # one page of one head, odd strides
    solo = torch.empty(1, 8, 1, 64, device="cuda", dtype=F16).copy_(solo).as_strided((1, 8, 1, 64), (3, 64, 5, 1))
    got = paged_attention(q[:1, :4], solo, solo, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), [8])
    _check(got, _reference(q[:1, :4], solo, solo, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), [8], [1]), F16,
           rounded=False)
    with pytest.raises(ValueError, match="k_pages must be 16-byte aligned"):
        paged_attention(q, k.transpose(2, 3).contiguous().transpose(2, 3), v, table, plan)


def test_page_numbers_are_clamped():
    """Page numbers outside the pool read its first or last page."""
    print("\n[case] page numbers outside the pool", flush=True)
    q, k, v, table, plan = _case([100, 90], [1, 1], [], 4, 2, 128, 8, BF)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    bad, good = table.clone(), table.clone()
    bad[0, 3], bad[1, 0], good[0, 3], good[1, 0] = -5, 1 << 30, 0, k.shape[0] - 1
    assert torch.equal(paged_attention(q, k, v, bad, plan), paged_attention(q, k, v, good, plan))


def test_falls_back_to_expressions():
    """float32 and other head_dims run the torch expressions; with gradients
    asked for, the call is differentiable."""
    print("\n[case] expressions on the GPU", flush=True)
    lens, new = [90, 33, 0], [2, 3, 1]
    for D, dtype in ((128, torch.float32), (96, BF), (32, F16)):
        q, k, v, table, plan = _case(lens, new, [], 6, 2, D, 8, dtype)
        ref = _reference(q, k, v, table, lens, new)
        _check(paged_attention(q, k, v, table, plan), ref, dtype)
    q, k, v, table, plan = _case(lens, new, [], 6, 2, 128, 8, torch.float32)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    w = torch.randn(q.shape, device="cuda")
    (paged_attention(*leaves, table, plan) * w).sum().backward()
    host = [t.detach().double().cpu().requires_grad_() for t in leaves]
    plan2 = PagedPlan(lens, heads=6, kv_heads=2, new_tokens=new, device="cpu")
    (paged_attention(*host, table.cpu(), plan2) * w.double().cpu()).sum().backward()
    for a, b in zip(leaves, host):
        # float32 gradients of sums over at most 90 tokens x 128 dims
        assert (a.grad.double().cpu() - b.grad).norm() <= 90 * 2.0 ** -24 * 16 * b.grad.norm()
    q = q.bfloat16().requires_grad_()
    assert paged_attention(q, k.bfloat16(), v.bfloat16(), table, plan).grad_fn is not None


def test_streams():
    """Calls run on the current stream, two at once from one plan and pools."""
    print("\n[case] two streams at once", flush=True)
    lens, new = [3000, 2000, 700], [1, 1, 1]
    q, k, v, table, plan = _case(lens, new, [([0, 1], 512)], 32, 8, 128, 16, BF)
    q2 = torch.randn_like(q)
    want, want2 = paged_attention(q, k, v, table, plan), paged_attention(q2, k, v, table, plan)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for s, x in ((s1, q), (s2, q2)):
            with torch.cuda.stream(s):
                got.append(paged_attention(x, k, v, table, plan))
    for s in (s1, s2):
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, want if i % 2 == 0 else want2) for i, g in enumerate(got))


def test_graph_replays():
    """A captured decode step, replayed with the plan updated between replays,
    gives the eager call's bits; the cache cannot change while capturing."""
    print("\n[case] captured append and attention, the plan updated between replays", flush=True)
    page, H, KVH, D = 8, 8, 2, 128
    cache = PagedKVCache(1, 200, page, kv_heads=KVH, head_dim=D, max_seqs=6, max_len=300)
    prompt, = cache.add([130])
    for t in (*cache.k, *cache.v):
        t.normal_()
    seqs = [prompt, *cache.fork(prompt, 3)]
    cache.extend(seqs, 1)
    plan = cache.plan(seqs, H, fixed=True)
    assert plan.prefixes == [([0, 1, 2, 3], 128)]
    g = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn(4, H + 2 * KVH, D, device="cuda", generator=g).bfloat16()
    cs = torch.randn(2, 4, D, device="cuda", generator=g).bfloat16()

    def step():
        q = rope_append(qkv, cs[0], cs[1], cache.k[0], cache.v[0], cache.block_table, plan)
        return paged_attention(q, cache.k[0], cache.v[0], cache.block_table, plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        for call in (lambda: cache.extend(seqs), lambda: cache.add([1]), lambda: cache.fork(prompt), cache.compact,
                     lambda: cache.free([prompt]), lambda: plan.update(plan.seq_lens)):
            with pytest.raises(RuntimeError, match="while a graph is captured"):
                call()
    for i in range(6):
        if i:
            cache.extend(seqs, [1, 17, 30, 2])
            plan.update(cache.lengths(seqs))
        qkv.normal_(generator=g)
        before = [t.clone() for t in (cache.k[0], cache.v[0])]
        graph.replay()
        got, k1, v1 = out.clone(), cache.k[0].clone(), cache.v[0].clone()
        cache.k[0].copy_(before[0])
        cache.v[0].copy_(before[1])
        torch.cuda.synchronize()
        eager = step()
        assert torch.equal(got, eager) and torch.equal(k1, cache.k[0]) and torch.equal(v1, cache.v[0])
        exact = paged_attention(got, cache.k[0], cache.v[0], cache.block_table, cache.plan(seqs, H))
        assert torch.isfinite(exact).all()


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype,D,H,KVH", [(BF, 128, 8, 2), (F16, 64, 7, 1), (BF, 16, 1, 1), (F16, 256, 2, 2)])
def test_rope_append(dtype, D, H, KVH):
    print(f"\n[case] rope append {dtype} D={D} H={H} KVH={KVH}", flush=True)
    lens, new = [70, 9, 130, 0, 2, 64], [3, 9, 1, 2, 4, 0]
    k, v, table = (t.cuda() for t in _shared_pools(lens, [], 8, KVH, D, 5, dtype=dtype))
    plan = PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new)
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn(plan.tokens, H + 2 * KVH, D, generator=g).to("cuda", dtype)
    cos, sin = (torch.randn(plan.tokens, D, generator=g).to("cuda", dtype) for _ in range(2))
    host = [t.cpu().clone() for t in (k, v)]
    q = rope_append(qkv, cos, sin, k, v, table, plan)
    plan2 = PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new, device="cpu")
    x, c, s = qkv.double(), cos.double()[:, None], sin.double()[:, None]
    want = x * c + torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1) * s
    # one rounding to the type, after two products and a sum in float32
    size = x.abs() * c.abs() + x.abs().roll(D // 2, -1) * s.abs()
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -22 * size + (2.0 ** -25 if dtype == F16 else 0)
    assert ((q.double() - want[:, :H]).abs() <= bound[:, :H]).all()
    rope_append(qkv.cpu(), cos.cpu(), sin.cpu(), *host, table.cpu(), plan2)
    # the CPU's expressions round the same float32 values, formed without fused multiply-adds
    step = 2 * torch.finfo(dtype).eps * host[0].double().abs() + 2.0 ** -20
    assert torch.equal(v.cpu().nan_to_num(9.0), host[1].nan_to_num(9.0))
    assert torch.equal(k.cpu().isnan(), host[0].isnan())
    assert ((k.cpu().double() - host[0].double()).abs().nan_to_num(0.0) <= step.nan_to_num(1.0)).all()
    written = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b, (n, t) in enumerate(zip(lens, new)):
        for pos in range(max(0, n - t), n):
            written[int(table[b, pos // 8]), pos % 8] = True
    before = _shared_pools(lens, [], 8, KVH, D, 5, dtype=dtype)
    assert torch.equal(k.cpu()[~written].nan_to_num(9.0), before[0][~written].nan_to_num(9.0))
    # pools interleaved in one tensor and a projection with odd strides
    both = torch.stack([before[0], before[1]], 1).cuda()
    wide = torch.zeros(plan.tokens, H + 2 * KVH + 1, D + 8, device="cuda", dtype=dtype)[:, 1:, 4:4 + D].copy_(qkv)
    assert torch.equal(rope_append(wide, cos, sin, both[:, 0], both[:, 1], table, plan), q)
    assert torch.equal(both[:, 0].nan_to_num(9.0), k.nan_to_num(9.0)) and torch.equal(both[:, 1].nan_to_num(9.0),
                                                                                      v.nan_to_num(9.0))
    with pytest.raises(ValueError, match="must not overlap"):
        rope_append(qkv, cos, sin, k[:1].expand(k.shape), v, table, plan)


# -------------------------------------------------------------------- pages
@pytest.mark.parametrize("seed", range(3))
def test_cache_matches_the_cpu(seed):
    """Random operations on a GPU cache and a CPU one leave the same block
    table and pools."""
    print(f"\n[case] cache operations, seed {seed}", flush=True)
    r = random.Random(seed)
    kw = dict(kv_heads=2, head_dim=24, max_seqs=7, max_len=900, dtype=F16)
    caches = [PagedKVCache(35, 700, 8, device=d, **kw) for d in ("cuda", "cpu")]
    for a, b in zip((*caches[0].k, *caches[0].v), (*caches[1].k, *caches[1].v)):
        b.normal_(generator=torch.Generator().manual_seed(seed))
        a.copy_(b)
    alive = []
    for _ in range(40):
        op = r.choice(("add", "extend", "extend", "fork", "free", "compact"))
        args = {"add": ([r.choice((0, 5, 8, 800)) for _ in range(r.randint(0, 2))],),
                "extend": (r.sample(alive, r.randint(0, len(alive))), r.choice((1, 3, 40))),
                "fork": (r.choice(alive) if alive else 0, r.randint(0, 3)),
                "free": (r.sample(alive, r.randint(0, len(alive))),), "compact": ()}[op]
        res = []
        for c in caches:
            try:
                res.append(getattr(c, op)(*args))
            except RuntimeError as e:
                res.append(str(e))
        assert res[0] == res[1]
        if op in ("add", "fork") and not isinstance(res[0], str):
            alive += res[0]
        if op == "free" and not isinstance(res[0], str):
            alive = [s for s in alive if s not in args[0]]
        for s in alive:
            n = len(caches[0].pages(s))
            assert caches[0].block_table[s, :n].tolist() == caches[0].pages(s) == caches[1].pages(s)
    for a, b in zip((*caches[0].k, *caches[0].v), (*caches[1].k, *caches[1].v)):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(caches[0].tables(alive[::-1]).cpu(), caches[0].block_table.cpu()[alive[::-1]])


def test_copy_pages():
    """More pools and pairs than one launch holds, pages of any size, views;
    captured copies run again in every replay."""
    print("\n[case] copy_pages", flush=True)
    g = torch.Generator().manual_seed(2)
    order = torch.randperm(1000, generator=g).tolist()
    src, dst = [order[i % 100] for i in range(900)], order[100:]
    for shape, n in (((1000, 8, 1, 8), 70), ((1000, 2, 3, 8), 3), ((1000, 40, 8, 16), 2)):
        pools = [torch.randn(shape, generator=g).bfloat16().cuda() for _ in range(n)]
        want = [t.clone() for t in pools]
        for t in want:
            t[torch.tensor(dst, device="cuda")] = t[torch.tensor(src, device="cuda")]
        copy_pages(pools, src, dst)
        assert all(torch.equal(a, b) for a, b in zip(pools, want))
    both = torch.randn(20, 2, 16, 64, generator=g).cuda()
    want = both.clone()
    want[[3, 4], 1] = want[[0, 0], 1]
    copy_pages(both[:, 1], [0, 0], [3, 4])
    assert torch.equal(both, want)
    x = torch.randn(6, 8, 8, generator=g).cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copy_pages(x, [0, 1], [4, 5])
    for _ in range(3):
        x.normal_()
        want = x.clone()
        want[[4, 5]] = want[[0, 1]]
        graph.replay()
        assert torch.equal(x, want)
    for s, d, text in [([0], [6], "no page"), ([0, 1], [2, 2], "written twice"), ([0, 1], [1, 2], "both read")]:
        with pytest.raises(RuntimeError, match=text):
            copy_pages(x, s, d)
    with pytest.raises(RuntimeError, match="16-byte"):
        copy_pages(torch.zeros(4, 3, device="cuda"), [0], [1])
    with pytest.raises(ValueError, match="host integers"):
        copy_pages(x, torch.tensor([0], device="cuda"), [1])


# -------------------------------------------------------------------- model
SMALL = LlamaShape(hidden=512, intermediate=1024, heads=4, kv_heads=1, layers=2, vocab=1000)


def test_copies_are_checked_before_any():
    """Pools of pages that are no whole 16-byte pieces are refused before the
    others' pages move."""
    print("\n[case] copies refused", flush=True)
    good = torch.arange(64, device="cuda").view(4, 16).float()
    before = good.clone()
    with pytest.raises(RuntimeError, match="16-byte"):
        copy_pages([good, torch.zeros(4, 3, device="cuda")], [0], [1])
    with pytest.raises(RuntimeError, match="16-byte"):
        copy_pages([good, torch.zeros(4 * 16 + 1, device="cuda")[1:].view(4, 16)], [0], [1])
    assert torch.equal(good, before)


@pytest.mark.parametrize("D, KVH, new", [(128, 8, [1, 1]), (64, 16, [5, 40])])
def test_offsets_past_32_bits(D, KVH, new):
    """Pages that lie more than 4 GiB, and 2^31 elements, from the pools' start:
    appended to, copied and attended to as in a small pool."""
    print(f"\n[case] large pools D={D}", flush=True)
    page, lens, H = 256, [900, 700], 4 * KVH
    few = sum(-(-n // page) for n in lens)
    num = (1 << 32) // (2 * page * KVH * D) + 2 * few  # K and V side by side: 8 GiB and some
    both = torch.empty(num, 2, page, KVH, D, dtype=BF, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    both[num - 2 * few:] = torch.randn(2 * few, 2, page, KVH, D, generator=g, device="cuda").bfloat16()
    small = both[num - 2 * few:].clone()
    q, qkv = (torch.randn(sum(new), n, D, generator=g, device="cuda").bfloat16() for n in (H, H + 2 * KVH))
    cs = torch.randn(2, sum(new), D, generator=g, device="cuda").bfloat16()
    order = torch.randperm(few, generator=torch.Generator().manual_seed(2))
    rows = torch.zeros(2, 4, dtype=torch.int32)
    rows[0, :4], rows[1, :3] = order[:4], order[4:7]
    got = []
    for pool, first in ((both, num - 2 * few), (small, 0)):
        table = (rows + first).cuda()
        plan = PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new)
        turned = rope_append(qkv, cs[0], cs[1], pool[:, 0], pool[:, 1], table, plan)
        copy_pages([pool.view(pool.shape[0], -1)], list(range(first, first + few)),
                   list(range(first + few, first + 2 * few)))
        got.append((turned, paged_attention(q, pool[:, 0], pool[:, 1], table, plan),
                    paged_attention(q, pool[:, 0], pool[:, 1], table + few, plan), pool[first:].clone()))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert torch.equal(got[0][1], got[0][2])
    _check(got[0][1], _reference(q, small[:, 0], small[:, 1], rows.cuda(), lens, new), BF)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_model_extends(dtype):
    """A prompt, samples of it with prompts of their own, decode steps and a
    compaction between them: the logits are those of each sequence prefilled by
    itself, to the tolerance of the runtime's decode against its prefill."""
    print(f"\n[case] model over a shared cache, {dtype}", flush=True)
    model = RandomLlama(SMALL, seed=11, std=0.05, device="cuda", dtype=dtype)
    g = torch.Generator().manual_seed(5)
    toks = torch.randint(0, SMALL.vocab, (6, 700), generator=g).cuda()
    toks[:, :400] = toks[0, :400]

    def check(logits, order, lens):
        for x, s in zip(logits, order):
            want = model.prefill(toks[s:s + 1, :lens[s]], NHDCache(SMALL, 1, lens[s], dtype, "cuda"))[0]
            assert (x - want).abs().max() <= 0.05 * want.abs().max()

    cache = _model_cache(SMALL, "cuda", dtype, num_pages=400, page_size=16, max_len=700)
    gone, first = cache.add([500, 0])
    check(model.extend(toks[:1, :400], cache, [first]), [0], [400])
    seqs = [first, *cache.fork(first, 5)]
    new = [1, 150, 40, 7, 64, 3]
    lens = [400 + n for n in new]
    packed = torch.cat([toks[s, 400:n] for s, n in enumerate(lens)])
    check(model.extend(packed, cache, seqs, new, mlp_chunk=100), range(6), lens)
    cache.free([gone])
    assert cache.compact() == cache.used_pages == 25 + sum(-(-n // 16) - 25 for n in lens)
    for i in range(3):
        logits = model.extend(torch.stack([toks[s, n] for s, n in enumerate(lens)]), cache, seqs, 1,
                              backend=ExactDecodeBackend() if i == 1 else None)
        lens = [n + 1 for n in lens]
        check(logits, range(6), lens)


def test_sampled_backends_read_the_cache():
    """santa_flash over the rows of a forked cache gives the bits it gives on the
    same tokens stored contiguously, also through the model."""
    print("\n[case] santa_flash over a forked cache", flush=True)
    backend = ab.build_backends(["santa_flash"], santa_s=128, santa_seed=3, santa_block_n=None, flashinfer_mode="auto",
                                flashinfer_use_tensor_cores=False)[0]
    cache = PagedKVCache(1, 300, 16, kv_heads=2, head_dim=128, max_seqs=4, max_len=1200)
    a, = cache.add([1000])
    cache.k[0].normal_()
    cache.v[0].normal_()
    b, = cache.fork(a)
    cache.extend([b], 37)
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    got = backend.decode_paged(q, cache.k[0], cache.v[0], cache.tables([b, a]), [1037, 1000])
    at = torch.arange(1037, device="cuda")
    flat = [torch.stack([t[cache.block_table[s, at.clamp_max(n - 1) // 16].long(), at.clamp_max(n - 1) % 16]
                         for s, n in ((b, 1037), (a, 1000))]) for t in (cache.k[0], cache.v[0])]
    want = backend._unwrap_tensor_out(backend.module.decode_systematic_batched(q, *flat, 128, seed=3,
                                                                               valid_len=[1037, 1000]))
    assert torch.equal(got, want)
    model = RandomLlama(SMALL, seed=1, std=0.05, device="cuda")
    held = _model_cache(SMALL, "cuda", BF, num_pages=100, page_size=16, max_len=600)
    s, = held.add([0])
    model.extend(torch.arange(300, device="cuda")[None], held, [s])
    logits = model.extend(torch.tensor([[5], [6]], device="cuda"), held, [s, *held.fork(s)], backend=backend)
    assert logits.shape == (2, SMALL.vocab) and torch.isfinite(logits).all() and backend.actual_mode == "paged"
