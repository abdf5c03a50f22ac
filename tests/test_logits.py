"""Rules on logits, on the CPU: against a formula in float64 written row by row,
gradients, and refusals."""
import ctypes
import math
import random

import pytest
import torch

from santa_amd import logits as L
from santa_amd.logits import adjust_logits
from santa_amd.paged import PagedPlan
from test_draft_trees import path, random_tree

# lens, new tokens, sequences without a tree (None: no trees), V, rows of the table
CASES = [
    ([5], [1], None, 7, None), ([0, 9, 30], [1, 1, 1], None, 33, [2, 0, 3]), ([40, 20], [6, 3], None, 100, None),
    ([40, 70, 6], [6, 1, 9], (), 129, [1, 4, 0]), ([128, 64, 20], [30, 64, 3], (2,), 64, None), ([8], [8], (), 1, None),
    ([300], [70], (), 2500, None),
]


def random_rules(g, r, V, S, N, K, kinds):
    """Rules of every kind, by sequence or for all."""
    rand = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    kw = {}
    if "repetition" in kinds:
        kw["repetition"] = rand(S) + 0.5 if r.random() < 0.6 else 1.3
    if "frequency" in kinds:
        kw["frequency"] = rand(S) - 0.3 if r.random() < 0.6 else 0.25
    if "presence" in kinds:
        kw["presence"] = rand(S) if r.random() < 0.6 else -0.5
    if "bias" in kinds:
        rows = r.choice((1, S))
        ids = torch.randint(-3, V + 3, (rows, K), generator=g, dtype=torch.int32)  # some twice, some of no token
        kw["bias"] = (ids, torch.randn(rows, K, generator=g) * 3)
    if "allowed" in kinds:
        rows = r.choice((1, N))
        kw["allowed"] = torch.randint(-(1 << 31), 1 << 31, (rows, -(-V // 32)), generator=g).to(torch.int32)
        if rows > 1:
            kw["allowed"][0] = 0  # a row that allows nothing
    if "prompts" in kinds:
        kw["prompts"] = torch.randint(0, 40, (S,), generator=g, dtype=torch.int32)
    return kw


ALL = ("repetition", "frequency", "presence", "bias", "allowed", "prompts")


def make(case, kinds=ALL, dtype=torch.float32, K=12, **plan_kw):
    lens, new, chains, V, rows = CASES[case]
    r, g = random.Random(case), torch.Generator().manual_seed(case)
    trees = None if chains is None else [None if b in chains else random_tree(r, t, 0.15) for b, t in enumerate(new)]
    S, N = 1 + max(rows or [len(lens) - 1]), sum(new)
    plan_kw = {"device": "cpu", **plan_kw}
    plan = PagedPlan(lens, heads=4, kv_heads=2, new_tokens=new, rows=rows, parents=trees, **plan_kw)
    logits = (torch.randn(N, V, generator=g) * 3).to(dtype)
    tokens = torch.randint(-1, V + 1, (S, max(lens) + 3), generator=g, dtype=torch.int32)
    tokens[:, ::2] = tokens[:, ::2] % min(V, 5)  # some often
    return logits, tokens, plan, random_rules(g, r, V, S, N, K, kinds)


def formula(logits, tokens, plan, repetition=1.0, frequency=0.0, presence=0.0, bias=None, allowed=None, prompts=None):
    """(values, sum of what is added up) in float64, row by row."""
    x, V = logits.double().clone(), logits.shape[1]
    size, r = x.abs(), 0
    of = lambda p, s: float(p[s]) if isinstance(p, torch.Tensor) else p  # noqa: E731
    for b, (s, n, t) in enumerate(zip(plan.rows, plan.seq_lens, plan.new_tokens)):
        parents = plan.parents[b] if plan.parents is not None else None
        for i in range(t):
            if parents is None:
                context, own = range(max(0, n - t + i + 1)), []
            elif n < t or parents[i] == -2:
                context, own = [], []
            else:
                context, own = range(n - t), [n - t + j for j in path(parents, i)]
            count, seen = {}, set()
            for p in [*context, *own] if tokens is not None else []:
                v = int(tokens[s, p])
                if 0 <= v < V:
                    seen.add(v)
                    if p in own or p >= (0 if prompts is None else int(prompts[s])):
                        count[v] = count.get(v, 0) + 1
            for v in seen:
                x[r, v] = x[r, v] / of(repetition, s) if x[r, v] > 0 else x[r, v] * of(repetition, s)
                size[r, v] = x[r, v].abs()
            for v, c in count.items():
                x[r, v] -= of(frequency, s) * c + of(presence, s)
                size[r, v] += abs(of(frequency, s)) * c + abs(of(presence, s))
            if bias is not None:
                last = {int(v): float(y) for v, y in zip(*(z[s if len(z) > 1 else 0] for z in bias)) if 0 <= int(v) < V}
                for v, y in last.items():
                    x[r, v] += y
                    size[r, v] += abs(y)
            if allowed is not None:
                bits = allowed[r if len(allowed) > 1 else 0].tolist()
                for v in range(V):
                    if not bits[v // 32] >> (v % 32) & 1:
                        x[r, v] = -math.inf
            r += 1
    return x, size


def check(out, want, roundings=5):
    """Five roundings at most (of the quotient, the count's product, two differences
    and a sum), each half a step of what is added up."""
    x, size = want
    assert out.dtype == torch.float32 and torch.equal(out == -math.inf, x == -math.inf)
    at = x > -math.inf
    assert ((out.double() - x).abs()[at] <= roundings * 2.0 ** -24 * size[at] + 1e-40).all()


@pytest.mark.parametrize("kinds", [ALL, ("repetition",), ("frequency", "prompts"), ("bias",), ("allowed",), ()])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_rules(case, kinds):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits, tokens, plan, kw = make(case, kinds, dtype)
        want = formula(logits, tokens, plan, **kw)
        out = adjust_logits(logits, tokens, plan, **kw)
        check(out, want)
        assert torch.equal(adjust_logits(logits, tokens.long(), plan, greedy=True, **kw), out.argmax(-1))
        none = {k: v for k, v in kw.items() if k != "prompts"}
        check(adjust_logits(logits, None, plan, **none), formula(logits, None, plan, **none))


def test_lengths_and_no_plan():
    logits, tokens, plan, kw = make(1)
    lens = [5, 20, 12, 9]
    x = torch.randn(4, 33)
    kw["allowed"] = kw["allowed"][:1]
    plan = PagedPlan(lens, heads=1, kv_heads=1, device="cpu")
    want = adjust_logits(x, tokens, plan, **kw)
    assert torch.equal(adjust_logits(x, tokens, lens, **kw), want)
    assert torch.equal(adjust_logits(x, tokens, torch.tensor(lens), **kw), want)
    bias = (torch.tensor([[3, -1], [4, 4], [99, -7], [0, 1]], dtype=torch.int32), torch.tensor([[1.0, 9], [2, 3], [4, 5], [6, 7]]))
    out = adjust_logits(x, bias=bias)
    x[0, 3] += 1
    x[1, 4] += 3
    x[3, 0] += 6
    x[3, 1] += 7
    assert torch.equal(out, x)
    assert adjust_logits(x[:0], greedy=True).shape == (0,) and adjust_logits(x[:0]).shape == (0, 33)
    assert torch.equal(adjust_logits(x, bias=(bias[0][:, :0], bias[1][:, :0])), x)


def test_not_finite():
    """NaN and infinities: masked ones do not show, others go through."""
    x = torch.tensor([[math.nan, 1.0, -math.inf, math.inf], [math.nan, 2.0, 3.0, 3.0], [-math.inf] * 4])
    bits = torch.tensor([[0b0110], [0b1110], [0b1111]], dtype=torch.int32)
    out = adjust_logits(x, torch.tensor([[0, 1, 2, 3]] * 3), [4, 2, 4], repetition=2.0, allowed=bits)
    assert out[0].tolist() == [-math.inf, 0.5, -math.inf, -math.inf] and out[1].tolist() == [-math.inf, 1.0, 3.0, 3.0]
    assert adjust_logits(x, greedy=True).tolist() == [0, 0, 0]
    assert adjust_logits(x, allowed=bits, greedy=True).tolist() == [1, 2, 0]
    assert adjust_logits(x, allowed=bits * 0, greedy=True).tolist() == [0, 0, 0]


def test_differentiates():
    logits, tokens, plan, kw = make(3, dtype=torch.float64)
    kw.pop("allowed")
    x = logits[:, :40].clone().requires_grad_()
    assert torch.autograd.gradcheck(lambda x: adjust_logits(x, tokens, plan, **kw), x)


def test_refusals():
    logits, tokens, plan, kw = make(3)
    N, V = logits.shape
    one = torch.ones(5)
    for args, more in [
        ((logits[0], tokens, plan), {}), ((logits.int(), tokens, plan), {}), ((logits[:, :0], tokens, plan), {}),
        ((logits, tokens), {}), ((logits[:-1], tokens, plan), {}), ((logits, tokens.float(), plan), {}),
        ((logits, tokens[:3], plan), {}), ((logits, tokens[:, :69], plan), {}), ((logits, tokens[0], plan), {}),
        ((logits, tokens, plan), {"prompts": torch.zeros(5)}), ((logits, tokens, plan), {"prompts": torch.zeros(4).int()}),
        ((logits, tokens, plan), {"repetition": 0.0}), ((logits, tokens, plan), {"repetition": math.inf}),
        ((logits, tokens, plan), {"repetition": one[:4]}), ((logits, tokens, plan), {"frequency": math.nan}),
        ((logits, tokens, plan), {"frequency": one.double()}), ((logits, tokens, plan), {"presence": one[None]}),
        ((logits,), {"bias": (torch.zeros(1, 3).int(), torch.zeros(1, 2))}),
        ((logits,), {"bias": (torch.zeros(1, 3), torch.zeros(1, 3))}),
        ((logits,), {"bias": (torch.zeros(1, 3).int(), torch.zeros(1, 3).double())}),
        ((logits,), {"bias": (torch.zeros(2, 3).int(), torch.zeros(2, 3))}),
        ((logits,), {"bias": (torch.zeros(3).int(), torch.zeros(3))}),
        ((logits,), {"bias": (torch.zeros(1, 2047).int(), torch.zeros(1, 2047))}),
        ((logits,), {"allowed": torch.zeros(1, 4).int()}), ((logits,), {"allowed": torch.zeros(1, 5)}),
        ((logits,), {"allowed": torch.zeros(2, 5).int()}), ((logits,), {"allowed": torch.zeros(5).int()}),
    ]:
        with pytest.raises(ValueError):
            adjust_logits(*args, **more)
    with pytest.raises(ValueError, match="are counted"):
        adjust_logits(torch.zeros(1, 3), torch.zeros(1, 1).long().expand(1, 1 << 19), [1 << 19])


def test_library_refusals():
    lib, info = L._lib(), PagedPlan([20, 9], heads=4, kv_heads=2, device="cpu")._info
    error = lambda: lib.santa_last_error().decode()  # noqa: E731
    one = ctypes.c_void_p(16)

    def call(x=one, dtype=2, stride=100, N=2, V=100, out=one, token=None, ws=one, size=1 << 20, plan=one, with_plan=True, **kw):
        rules = L._Rules(**{"tokens": 16, "tokens_rows": 2, "tokens_len": 20, "tokens_stride": 20, **kw})
        return lib.santa_adjust_logits(x, dtype, stride, N, V, ctypes.byref(rules), ctypes.byref(info) if with_plan else None,
                                       plan, out, token, ws, size, None)

    for kw, text in [({"x": None}, "bad adjust"), ({"V": 0}, "bad adjust"), ({"V": 101}, "bad adjust"), ({"N": -1}, "bad adjust"),
                     ({"out": None}, "bad adjust"), ({"token": one}, "bad adjust"), ({"plan": None}, "bad adjust"),
                     ({"dtype": 3}, "bf16, f16 or float32"), ({"N": 3}, "the plan is for 2"), ({"tokens_rows": 1}, "row 1"),
                     ({"tokens_len": 19}, "token 19"), ({"with_plan": False}, "a plan says"), ({"tokens": 18}, "aligned"),
                     ({"biases": 3}, "bad adjust"), ({"biases": 2047, "bias_ids": 16, "bias": 16}, "up to 2046"),
                     ({"out": None, "token": one, "size": 7}, "workspace"), ({"out": None, "token": one, "ws": None}, "workspace")]:
        assert call(**kw) != 0 and text in error(), (kw, error())
    assert lib.santa_adjust_logits_workspace_size(4, 128256, 4) >= 32 and lib.santa_adjust_logits_workspace_size(0, 5, 0) == 0
