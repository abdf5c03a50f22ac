"""Rules on logits, on the CPU, at the edges of what a call may say."""
import ctypes

import pytest
import torch

from santa_amd import logits as L
from santa_amd.logits import adjust_logits
from santa_amd.paged import PagedPlan


@pytest.mark.parametrize("kw", [{"repetition": 2.0}, {"frequency": 0.5}, {"presence": -0.5}, {"repetition": torch.ones(3)},
                                {"frequency": torch.zeros(3)}, {"prompts": torch.zeros(3, dtype=torch.int32)}])
def test_penalties_without_tokens(kw):
    """A call that forgot the tokens is refused, where it gave the logits back."""
    x = torch.randn(3, 9)
    with pytest.raises(ValueError, match="without tokens there are none"):
        adjust_logits(x, **kw)
    with pytest.raises(ValueError, match="without tokens there are none"):
        adjust_logits(x, greedy=True, **kw)
    assert torch.equal(adjust_logits(x, repetition=1.0, frequency=0.0, presence=-0.0), x)
    assert torch.equal(adjust_logits(x, None, [4, 5, 6], **kw), x)  # a plan, whose rows have seen none


def under_vmap(device):
    """What is mapped alone -> (values, those of calls one by one)."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 40, generator=g).to(device)
    i = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, dtype=torch.int64).to(torch.int32).to(device)  # noqa: E731
    tokens, prompts, ids, bits = i(0, 40, 2, 3, 6), i(0, 6, 2, 3), i(-1, 41, 2, 3, 4), i(-(1 << 31), 1 << 31, 2, 3, 2)
    values, lens = torch.randn(2, 3, 4, generator=g).to(device), [4, 5, 6]
    penalties = torch.rand(2, 3, generator=g).to(device) + 0.5
    calls = {
        "logits": (torch.stack([x, -x]), lambda y: adjust_logits(y, tokens[0], lens, repetition=2.0)),
        "tokens": (tokens, lambda t: adjust_logits(x, t, lens, repetition=2.0, frequency=0.5)),
        "prompts": (prompts, lambda p: adjust_logits(x, tokens[0], lens, prompts=p, frequency=0.5)),
        "ids": (ids, lambda b: adjust_logits(x, bias=(b, values[0]))),
        "values": (values, lambda b: adjust_logits(x, bias=(ids[0], b))),
        "allowed": (bits, lambda b: adjust_logits(x, allowed=b)),
        "penalty": (penalties, lambda p: adjust_logits(x, tokens[0], lens, repetition=p)),
        "tree": (tokens, lambda t: adjust_logits(x, t, _tree(device), presence=0.5)),
        "token": (bits, lambda b: adjust_logits(x, allowed=b, greedy=True)),
    }
    return {k: (torch.vmap(f)(mapped), torch.stack([f(y) for y in mapped])) for k, (mapped, f) in calls.items()}


def _tree(device):
    return PagedPlan([6], heads=1, kv_heads=1, new_tokens=[3], parents=[[-1, 0, 0]], device=device)


def test_vmap():
    """Under vmap over one argument alone, whichever it is, a call gives what it
    gives for each."""
    for what, (out, want) in under_vmap("cpu").items():
        assert torch.equal(out, want), what


def test_library_refuses_what_is_not_aligned():
    """The plan, which kernels read in pairs, and every array of the call."""
    lib, info = L._lib(), PagedPlan([20, 9], heads=4, kv_heads=2, device="cpu")._info

    def call(x=4096, dtype=2, plan=4096, out=4096, token=None, **kw):
        rules = L._Rules(**{"tokens": 4096, "tokens_rows": 2, "tokens_len": 20, "tokens_stride": 20, "biases": 3,
                            "bias_ids": 4096, "bias": 4096, **kw})
        rc = lib.santa_adjust_logits(x, dtype, 100, 2, 100, ctypes.byref(rules), ctypes.byref(info), plan, out, token,
                                     4096, 0, None)
        assert rc != 0
        return lib.santa_last_error().decode()

    for off in (4, 8):  # without it the refusal is the one of the workspace, which comes last
        assert "the plan must be 16-byte aligned" in call(plan=4096 + off, out=None, token=4096)
    assert "workspace" in call(out=None, token=4096)
    for kw in ({"x": 4098}, {"x": 4097, "dtype": 0}, {"out": 4098}, {"out": None, "token": 4100}):
        assert "aligned to their elements" in call(**kw)
    for name in ("prompts", "repetition", "frequency", "presence", "bias_ids", "bias", "allowed"):
        assert "rules' arrays" in call(out=None, token=4096, **{name: 4098})
    assert "aligned" in call(out=None, token=4096, tokens=4100, tokens_wide=1)
