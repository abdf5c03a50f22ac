"""Rotary tables and the norms and rotations of rope_append on the GPU, against
float64.

Tolerances.  Tables: the angle's part of a turn is rounded to float32 (2^-25 of at
most half a turn: 2 pi 2^-26 of 1) and so are cos and sin (sincospif: 4 steps of
2^-24 at most), then the table's own rounding (eps, half a step).  Heads: the mean of
D squares is off by at most (D + 2) steps of 2^-24 of itself, its root's inverse by
half of that and 2 more, the products with the weight, cos and sin and their sum by one
each; all relative to |x c| + |other s|, and the result is rounded once.

Every case prints its name before touching the GPU.
"""
import math

import pytest
import torch

from santa_amd.paged import PagedPlan, RopeScaling, rope_append, rope_tables
from test_paged import _shared_pools
from test_rotary import SCALINGS, append, tables

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("dim, interleaved", [(128, False), (128, True), (64, False), (6, True), (2, False), (182, False),
                                              (512, True), (20, False)])
def test_tables(dim, interleaved, dtype):
    print(f"\n[case] tables dim={dim} interleaved={interleaved} {dtype}", flush=True)
    scalings = [s for s in SCALINGS if dim > 2 or s is None or s.kind != "ntk"]
    for j, scaling in enumerate(scalings):
        pos = [0, 1, 77, 8191, 131071, 2000003, -1, 4000][:8 if j else 7]
        want = tables(pos, dim, 10000.0, scaling, interleaved)
        for at in (torch.tensor(pos).cuda(), torch.tensor(pos, dtype=torch.int32).cuda(),
                   torch.tensor([[p, 5] for p in pos], dtype=torch.int32).cuda()[:, 0]):
            got = rope_tables(at, dim, scaling=scaling, interleaved=interleaved, dtype=dtype)
            for a, b in zip(got, want):
                eps = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
                up = 1.0 if scaling is None or scaling.kind != "yarn" else 1.3
                off = up * (2 * math.pi * 2.0 ** -26 + 5 * 2.0 ** -24 + 2e6 * 2.0 ** -50)
                assert a.dtype == dtype and ((a.double().cpu() - b).abs() <= eps * b.abs() + off).all()


def test_tables_of_many_positions():
    print("\n[case] many positions; none; more dims than the kernel takes", flush=True)
    pos = torch.randint(0, 1 << 20, (30011,), device="cuda")
    for dim in (128, 600):
        for scaling in (None, RopeScaling("yarn", 4.0)):
            for dtype in (BF, torch.float64):
                a = rope_tables(pos, dim, scaling=scaling, dtype=dtype)
                b = rope_tables(pos.cpu(), dim, scaling=scaling, dtype=torch.float64)
                for x, y in zip(a, b):
                    y = y.cuda()
                    bound = 2.0 ** -8 * y.abs() + 1e-6 if dtype == BF else 1e-9
                    assert ((x.double() - y).abs() <= bound).all()
    assert rope_tables(pos[:0], 128)[0].shape == (0, 128)


def _bound(qkv, cos, sin, H, KVH, q_norm, k_norm, eps, interleaved, dtype, want):
    """Elementwise bounds of the rotated heads [N, H + KVH, D]."""
    x, D, R = qkv.double()[:, :H + KVH].abs(), qkv.shape[2], cos.shape[1]
    if q_norm is not None or k_norm is not None:
        n = x / torch.sqrt(qkv.double()[:, :H + KVH].square().mean(-1, keepdim=True) + eps)
        parts = ((slice(0, H), q_norm), (slice(H, H + KVH), k_norm))
        x = torch.cat([x[:, at] if w is None else n[:, at] * w.double().abs() for at, w in parts], 1)
    y, c, s = x[..., :R], cos.double().abs()[:, None], sin.double().abs()[:, None]
    if interleaved:
        other = torch.stack([y[..., 1::2], y[..., ::2]], -1).flatten(-2)
    else:
        other = torch.cat([y[..., R // 2:], y[..., :R // 2]], -1)
    size = torch.cat([y * c + other * s, x[..., R:]], -1)
    half = torch.finfo(dtype).eps / 2
    off = (D / 2 + 10) * 2.0 ** -24 * size * (1 + half) + half * want.abs()
    return off + 2.0 ** -25 if dtype == F16 else off


CASES = [
    # D, R, H, KVH, norms, interleaved, dtype
    (128, 128, 8, 2, "both", False, BF), (128, 64, 8, 2, "both", True, BF), (128, 32, 7, 1, "per head", False, F16),
    (128, 128, 4, 4, "none", True, BF), (64, 64, 12, 1, "q", False, F16), (64, 16, 4, 2, "k", True, BF),
    (128, 24, 4, 2, "both", False, BF),   # halves that are no whole pieces
    (128, 24, 4, 2, "both", True, F16), (128, 6, 4, 2, "none", False, BF), (64, 62, 4, 2, "per head", True, BF),
    (16, 16, 2, 1, "both", False, BF), (32, 8, 2, 1, "both", True, F16), (48, 48, 3, 3, "both", False, BF),
    (80, 32, 2, 1, "per head", False, F16), (256, 64, 4, 2, "both", False, BF), (512, 512, 2, 1, "both", True, BF),
    (96, 96, 2, 1, "q", True, BF), (272, 2, 2, 1, "k", False, F16), (16, 8, 2, 2, "both", False, BF),
    (256, 200, 2, 1, "per head", False, F16),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_append(case):
    D, R, H, KVH, norms, interleaved, dtype = CASES[case]
    print(f"\n[case] append D={D} R={R} H={H} KVH={KVH} {norms} interleaved={interleaved} {dtype}", flush=True)
    lens, new, page = [100, 17, 3, 60], [40, 1, 5, 0], 16
    k, v, table = (t.cuda() for t in _shared_pools(lens, [], page, KVH, D, case, dtype=dtype))
    k, v = k.nan_to_num(0.25), v.nan_to_num(0.25)
    g = torch.Generator(device="cuda").manual_seed(case)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    qkv, cos, sin = r(46, H + 2 * KVH, D), r(46, R), r(46, R)
    qkv[3, 1] = 0  # a head of zeros: eps alone under the root
    q_norm = {"q": r(D), "both": r(D), "per head": r(H, D)}.get(norms)
    k_norm = {"k": r(D), "both": r(D), "per head": r(KVH, D)}.get(norms)
    plan = PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new)
    host = [t.cpu() for t in (qkv, cos, sin, k, v, table)]
    want = append(*host, lens, new, H, *(w if w is None else w.cpu() for w in (q_norm, k_norm)), 1e-5, interleaved)
    kw = dict(q_norm=q_norm, k_norm=k_norm, eps=1e-5, interleaved=interleaved)
    k2, v2 = k.clone(), v.clone()
    q = rope_append(qkv, cos, sin, k2, v2, table, plan, **kw)
    assert torch.equal(v2.cpu().double(), want[2])
    rotated = torch.cat([want[0], torch.zeros(46, KVH, D, dtype=torch.float64)], 1)
    rows = [(b, n - t + i, t0 + i) for b, (n, t, t0) in enumerate(zip(lens, new, (0, 40, 41, 46)))
            for i in range(max(0, t - n), t)]
    for b, p, t in rows:
        rotated[t, H:] = want[1][host[5][b, p // page].long(), p % page]
    got = torch.zeros_like(rotated)
    got[:, :H] = q.cpu().double()
    left = k2.clone()
    for b, p, t in rows:
        at = (host[5][b, p // page].long(), p % page)
        got[t, H:] = k2[at].cpu().double()
        left[at] = k[at]
    assert torch.equal(left, k)  # nothing else was written
    bound = _bound(qkv, cos, sin, H, KVH, q_norm, k_norm, 1e-5, interleaved, dtype, rotated.cuda()).cpu()
    assert torch.isfinite(got).all() and ((got - rotated).abs() <= bound).all()
    # views of larger tensors, and weights that are not packed
    wide = torch.stack([qkv, qkv], 2)[:, :, 0]
    both = torch.stack([k, v], 1)
    kw.update((name, torch.stack([w, w], -1)[..., 0]) for name, w in (("q_norm", q_norm), ("k_norm", k_norm)) if w is not None)
    assert torch.equal(rope_append(wide, cos, sin, both[:, 0], both[:, 1], table, plan, **kw), q)
    assert torch.equal(both[:, 0], k2) and torch.equal(both[:, 1], v2)


def test_defaults_are_the_plain_rotation():
    """Without norms, over the whole head in halves: one kernel, whatever eps is."""
    print("\n[case] plain rotation", flush=True)
    k, v, table = (t.cuda() for t in _shared_pools([30], [], 16, 2, 128, 0, dtype=BF))
    plan = PagedPlan([30], heads=4, kv_heads=2, new_tokens=7)
    qkv, cos, sin = torch.randn(7, 8, 128).cuda().to(BF), torch.randn(7, 128).cuda().to(BF), torch.randn(7, 128).cuda().to(BF)
    a = rope_append(qkv, cos, sin, k.clone(), v.clone(), table, plan)
    b = rope_append(qkv, cos, sin, k.clone(), v.clone(), table, plan, eps=0.5, interleaved=False)
    assert torch.equal(a, b)


def test_autograd_takes_the_expressions():
    print("\n[case] autograd", flush=True)
    k, v, table = (t.cuda() for t in _shared_pools([30], [], 16, 2, 16, 0, dtype=BF))
    plan = PagedPlan([30], heads=4, kv_heads=2, new_tokens=7)
    qkv, cs, w = torch.randn(7, 8, 16).cuda().to(BF), torch.randn(7, 16).cuda().to(BF), torch.ones(16).cuda().to(BF)
    w.requires_grad_()
    q = rope_append(qkv, cs, cs, k, v, table, plan, q_norm=w)
    assert torch.autograd.grad(q.float().sum(), w)[0].abs().sum() > 0


def test_streams_and_replays():
    """On a stream of its own, and captured: the tables of a fixed tree plan and the
    append follow its updates."""
    print("\n[case] streams and replays", flush=True)
    lens, D, trees = [200, 90], 64, [[-1, 0, 0, 1], [-1, -1, 0]]
    k, v, table = (t.cuda() for t in _shared_pools([300, 300], [], 16, 2, D, 0, dtype=BF))
    k, v = k.nan_to_num(0.25), v.nan_to_num(0.25)
    plan = PagedPlan(lens, heads=4, kv_heads=2, new_tokens=[4, 3], parents=trees, fixed=True)
    qkv, w = torch.randn(7, 8, D).cuda().to(BF), torch.rand(D).cuda().to(BF)

    def call(k, v, plan):
        cos, sin = rope_tables(plan.positions, 32, scaling=RopeScaling("llama3", 8.0), interleaved=True)
        return rope_append(qkv, cos, sin, k, v, table, plan, q_norm=w, k_norm=w, interleaved=True)

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        k1, v1 = k.clone(), v.clone()
        q1 = call(k1, v1, plan)
    side.synchronize()
    kc, vc = k.clone(), v.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = call(kc, vc, plan)
    for n, other in ((lens, None), ([64, 300], [[-1, 0, 1, 2], [-1, -2, 0]]), ([300, 2], [[-1, -1, -1, 0], [-1, 0, 0]])):
        plan.update(n, other)
        kc.copy_(k), vc.copy_(v)
        qkv.copy_(torch.randn_like(qkv) if n is not lens else qkv)
        graph.replay()
        torch.cuda.synchronize()
        k2, v2 = k.clone(), v.clone()
        fresh = PagedPlan(n, heads=4, kv_heads=2, new_tokens=[4, 3], parents=plan.parents)
        q2 = call(k2, v2, fresh)
        assert torch.equal(q, q2) and torch.equal(kc, k2) and torch.equal(vc, v2)
        if n is lens:
            assert torch.equal(q1, q2) and torch.equal(k1, k2) and torch.equal(v1, v2)
