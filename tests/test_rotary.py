"""Rotary tables and the norms and rotations of rope_append on the CPU: against
formulas in float64 written head by head, gradients, and refusals."""
import ctypes
import math

import pytest
import torch

from santa_amd import paged
from santa_amd.paged import PagedPlan, RopeScaling, rope_append, rope_tables
from test_paged import _shared_pools

SCALINGS = [None, RopeScaling("linear", 4.0), RopeScaling("ntk", 3.0), RopeScaling("llama3", 8.0),
            RopeScaling("llama3", 32.0, 4096, low=0.5, high=7.0), RopeScaling("yarn", 16.0, 4096),
            RopeScaling("yarn", 4.0, 2048, low=2.0, high=20.0, magnitude=0.7)]


def frequency(i, dim, theta, s):
    """(angle per position of pair i, magnitude), from the published rules."""
    if s is None:
        return theta ** (-2 * i / dim), 1.0
    if s.kind == "ntk":
        return (theta * s.factor ** (dim / (dim - 2))) ** (-2 * i / dim), 1.0
    f = theta ** (-2 * i / dim)
    if s.kind == "linear":
        return f / s.factor, 1.0
    low, high = s.low or 1.0, s.high or (4.0 if s.kind == "llama3" else 32.0)
    if s.kind == "llama3":
        wave = 2 * math.pi / f
        if wave < s.original_len / high:
            return f, 1.0
        if wave > s.original_len / low:
            return f / s.factor, 1.0
        smooth = (s.original_len / wave - low) / (high - low)
        return (1 - smooth) * f / s.factor + smooth * f, 1.0
    pair = lambda turns: dim * math.log(s.original_len / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    first, last = max(0, math.floor(pair(high))), min(dim - 1, math.ceil(pair(low)))
    ramp = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
    return f / s.factor * ramp + f * (1 - ramp), 0.1 * math.log(s.factor) + 1 if s.magnitude is None else s.magnitude


def tables(pos, dim, theta, scaling, interleaved):
    cos, sin = (torch.zeros(len(pos), dim, dtype=torch.float64) for _ in range(2))
    for i in range(dim // 2):
        f, up = frequency(i, dim, theta, scaling)
        for d in ((2 * i, 2 * i + 1) if interleaved else (i, i + dim // 2)):
            for n, p in enumerate(pos):
                cos[n, d], sin[n, d] = up * math.cos(p * f), up * math.sin(p * f)
    return cos, sin


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scaling", SCALINGS)
def test_tables(scaling, interleaved):
    pos = [0, 1, 5, 8191, 8192, 131071, 2000003, -1]
    for dim, theta in ((64, 10000.0), (128, 500000.0), (6, 10000.0)):
        want = tables(pos, dim, theta, scaling, interleaved)
        for dtype in (torch.int32, torch.int64):
            got = rope_tables(torch.tensor(pos, dtype=dtype), dim, theta=theta, scaling=scaling, interleaved=interleaved,
                              dtype=torch.float64)
            # an angle of up to 2e6 is off by half a step (2^-33), as is the frequency under it
            assert all((a - b).abs().max() < 2e6 * 2.0 ** -50 for a, b in zip(got, want))
        got = rope_tables(torch.tensor(pos), dim, theta=theta, scaling=scaling, interleaved=interleaved)
        assert all(a.dtype == torch.bfloat16 and ((a - b).abs() <= 2.0 ** -8 * b.abs() + 1e-8).all()
                   for a, b in zip(got, want))
    empty = rope_tables(torch.zeros(0, dtype=torch.int32), 8, scaling=scaling)
    assert empty[0].shape == empty[1].shape == (0, 8)


def test_positions_of_a_plan():
    plan = PagedPlan([20, 9], heads=2, kv_heads=1, new_tokens=[3, 2], device="cpu", parents=[[-1, 0, 0], None])
    assert plan.positions.tolist() == [17, 18, 18, 7, 8]
    want = tables([17, 18, 18, 7, 8], 8, 10000.0, None, False)
    assert all(torch.allclose(a, b) for a, b in zip(rope_tables(plan.positions, 8, dtype=torch.float64), want))


def append(qkv, cos, sin, k, v, table, lens, new, H, q_norm, k_norm, eps, interleaved):
    """Head by head in float64: (q, k pages, v pages)."""
    N, KVH, D, R, page = len(qkv), k.shape[2], qkv.shape[2], cos.shape[1], k.shape[1]
    x, c, s = qkv.double().clone(), cos.double(), sin.double()
    y = x.clone()
    for h in range(H + KVH):
        w = q_norm if h < H else k_norm
        if w is not None:
            w = w.double().view(-1, D)
            w = w[(h if h < H else h - H) if len(w) > 1 else 0]
            x[:, h] = x[:, h] / torch.sqrt(x[:, h].square().sum(-1, keepdim=True) / D + eps) * w
        y[:, h] = x[:, h]
        for i in range(R // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
            y[:, h, a] = x[:, h, a] * c[:, a] - x[:, h, b] * s[:, a]
            y[:, h, b] = x[:, h, b] * c[:, b] + x[:, h, a] * s[:, b]
    k, v, t0 = k.double().clone(), v.double().clone(), 0
    for b, (n, t) in enumerate(zip(lens, new)):
        for i in range(max(0, t - n), t):
            at = (table[b, (n - t + i) // page].long(), (n - t + i) % page)
            k[at], v[at] = y[t0 + i, H:H + KVH], x[t0 + i, H + KVH:]
        t0 += t
    return y[:, :H], k, v


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norms", ["none", "q", "k", "both", "per head"])
@pytest.mark.parametrize("D, R", [(16, 16), (16, 6), (6, 2), (48, 32)])
def test_append(D, R, norms, interleaved):
    lens, new, H, KVH = [20, 9, 2], [3, 1, 4], 4, 2
    k, v, table = (t.nan_to_num(0.0) if t.is_floating_point() else t for t in _shared_pools(lens, [], 8, KVH, D, R))
    g = torch.Generator().manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    qkv, cos, sin = r(8, H + 2 * KVH, D), r(8, R), r(8, R)
    q_norm = {"q": r(D), "both": r(D), "per head": r(H, D)}.get(norms)
    k_norm = {"k": r(D), "both": r(D), "per head": r(KVH, D)}.get(norms)
    plan = PagedPlan(lens, heads=H, kv_heads=KVH, new_tokens=new, device="cpu")
    want = append(qkv, cos, sin, k, v, table, lens, new, H, q_norm, k_norm, 0.01, interleaved)
    q = rope_append(qkv, cos, sin, k, v, table, plan, q_norm=q_norm, k_norm=k_norm, eps=0.01, interleaved=interleaved)
    assert all((a - b).abs().max() < 1e-12 for a, b in zip((q, k, v), want))


def test_append_differentiates():
    k, v, table = (t.nan_to_num(0.0) if t.is_floating_point() else t for t in _shared_pools([9], [], 8, 1, 4, 1))
    plan = PagedPlan([9], heads=2, kv_heads=1, new_tokens=2, device="cpu")
    leaves = [torch.randn(*s, dtype=torch.float64).requires_grad_() for s in ((2, 4, 4), (2, 2), (2, 2), (2, 4), (4,))]

    def f(qkv, cos, sin, q_norm, k_norm):
        k2, v2 = k.clone(), v.clone()
        q = rope_append(qkv, cos, sin, k2, v2, table, plan, q_norm=q_norm, k_norm=k_norm, interleaved=True)
        return q, k2, v2

    assert torch.autograd.gradcheck(f, leaves)


def test_refusals():
    k, v, table = _shared_pools([20, 9], [], 8, 2, 16, 1)
    plan = PagedPlan([20, 9], heads=4, kv_heads=2, device="cpu")
    qkv, cs, w = (torch.zeros(*s, dtype=torch.float64) for s in ((2, 8, 16), (2, 16), (16,)))
    for args, kw in [((cs[:, :5], cs[:, :5]), {}), ((cs[:, :0], cs[:, :0]), {}), ((cs, cs[:, :8]), {}),
                     ((torch.cat([cs, cs], 1),) * 2, {}), ((cs[0], cs[0]), {}), ((cs, cs), {"q_norm": w[:8]}),
                     ((cs, cs), {"q_norm": w.expand(2, 16)}), ((cs, cs), {"k_norm": w.expand(4, 16)}),
                     ((cs, cs), {"k_norm": w.float()}), ((cs, cs), {"q_norm": w, "eps": -1.0}),
                     ((cs, cs), {"q_norm": w, "eps": math.nan})]:
        with pytest.raises(ValueError):
            rope_append(qkv, *args, k, v, table, plan, **kw)
    p = torch.arange(3)
    for args, kw in [((p.float(), 8), {}), ((p[None], 8), {}), ((p, 7), {}), ((p, 0), {}), ((p, 8), {"theta": 1.0}),
                     ((p, 8), {"theta": math.nan}), ((p, 8), {"dtype": torch.int32}),
                     ((p, 2), {"scaling": RopeScaling("ntk", 2.0)})]:
        with pytest.raises(ValueError):
            rope_tables(*args, **kw)
    for kw in ({"kind": "other", "factor": 2.0}, {"kind": "yarn", "factor": 0.0}, {"kind": "yarn", "factor": math.nan},
               {"kind": "llama3", "factor": 2.0, "low": 5.0}, {"kind": "linear", "factor": 2.0, "original_len": 0},
               {"kind": "yarn", "factor": 2.0, "magnitude": math.inf}):
        with pytest.raises(ValueError):
            RopeScaling(**kw)


def test_library_refusals():
    lib = paged._lib()
    error = lambda: lib.santa_last_error().decode()  # noqa: E731
    one, turns = ctypes.c_void_p(16), (ctypes.c_double * 300)()

    def table(pos=one, n=3, pairs=4, dtype=0, cos=one):
        return lib.santa_rope_tables(pos, 0, 1, n, turns, pairs, 1.0, 0, dtype, cos, one, None)

    for kw, text in [({"pos": None}, "bad rope_tables"), ({"n": -1}, "bad rope_tables"), ({"pairs": 0}, "bad rope_tables"),
                     ({"cos": None}, "bad rope_tables"), ({"dtype": 3}, "float32"), ({"pairs": 257}, "up to 512"),
                     ({"n": 1 << 40}, "too many")]:
        assert table(**kw) != 0 and text in error(), kw
    assert table(n=0, pos=None, cos=None) == 0
    plan = PagedPlan([20, 9], heads=4, kv_heads=2, device="cpu")
    strides = (ctypes.c_longlong * 6)(2048, 256, 128, 2048, 256, 128)

    def append(cos=one, R=128, qn=None, qh=1, kn=None, kh=1, eps=0.0, D=128, page=8):
        return lib.santa_paged_heads_append(one, cos, one, R, 0, qn, qh, kn, kh, eps, one, one, one, 0, D, 4, page, strides,
                                            one, 4, 2, ctypes.byref(plan._info), one, None)

    for kw, text in [({"cos": None}, "bad heads_append"), ({"cos": ctypes.c_void_p(8)}, "16-byte"),
                     ({"qn": ctypes.c_void_p(8)}, "16-byte"), ({"R": 129}, "even"), ({"R": 130}, "even"), ({"R": 0}, "even"),
                     ({"D": 520}, "up to 512"), ({"D": 528}, "up to 512"), ({"qn": one, "qh": 2}, "one per head"),
                     ({"kn": one, "kh": 4}, "one per head"), ({"eps": -1.0}, "eps"), ({"eps": math.nan}, "eps"),
                     ({"page": 12}, "power of two")]:
        assert append(**kw) != 0 and text in error(), (kw, error())
