"""Rules on logits on the GPU where their values are out of the ordinary: bit for bit
against the expressions on the CPU, NaN for NaN.  Every case prints its name before
touching the GPU."""
import math
import random

import pytest
import torch

from santa_amd.logits import adjust_logits
from santa_amd.paged import PagedPlan
from test_draft_trees import random_tree
from test_logits_edges import under_vmap
from test_logits_gpu import cuda, same

pytestmark = pytest.mark.gpu


def alike(out, want):
    return torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("what", ["repetition", "frequency", "presence"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, 3e38])
def test_penalties_that_are_not_finite(what, value):
    """They reach the tokens that they are for: those of the answer, or all that the
    row has seen; not those of the prompt, of a bias or of no rule."""
    print(f"\n[case] {what} {value}", flush=True)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 50, generator=g)
    tokens = torch.tensor([[1, 2, 2, 3, 4, 4], [5, 6, 7, 8, 9, 9], [0, 0, 0, 0, 0, 0]], dtype=torch.int32)
    kw = {what: torch.tensor([value, 1.5, value]), "prompts": torch.tensor([3, 2, 6], dtype=torch.int32),
          "bias": (torch.tensor([[1, 10, 4]], dtype=torch.int32), torch.tensor([[0.5, -1.0, 2.0]]))}
    want = adjust_logits(x, tokens, [6, 6, 5], **kw)
    out = adjust_logits(x.cuda(), tokens.cuda(), [6, 6, 5], **{k: cuda(v) for k, v in kw.items()})
    assert alike(out.cpu(), want)
    if what != "repetition" and not math.isfinite(value):  # of the third row all tokens are the prompt's
        assert torch.isfinite(want[2]).all() and torch.isfinite(want[0, [1, 2, 10]]).all()
        assert not torch.isfinite(want[0, 3])


def test_any_nan():
    """A bias or a penalty of any NaN gives one, with whatever bits."""
    print("\n[case] NaN of any bits", flush=True)
    nans = torch.tensor([0x7fc0feed, 0x7fc00000, -1, 0x7f800001], dtype=torch.int32).view(torch.float32)
    x, ids = torch.randn(4, 9), torch.tensor([[5]] * 4, dtype=torch.int32)
    tokens = torch.tensor([[2, 2]] * 4, dtype=torch.int32)
    want = x.clone()
    want[:, 5] = math.nan
    out = adjust_logits(x.cuda(), bias=(ids.cuda(), nans[:, None].cuda()))
    assert alike(out.cpu(), want)
    for name in ("repetition", "frequency", "presence"):
        want = x.clone()
        want[:, 2] = math.nan
        assert alike(adjust_logits(x.cuda(), tokens.cuda(), [2] * 4, **{name: nans.cuda()}).cpu(), want)
    x[:, 5] = nans  # of the logits themselves, with a rule and without
    want = x.clone()
    assert alike(adjust_logits(x.cuda()).cpu(), want)
    assert alike(adjust_logits(x.cuda(), bias=(ids.cuda(), torch.ones(4, 1).cuda())).cpu(), want)
    assert adjust_logits(x.cuda(), greedy=True).tolist() == [5] * 4


def test_vmap():
    """Tensors that a transform wraps have no memory for a kernel to read: whichever
    argument it is alone, the expressions take it."""
    print("\n[case] vmap", flush=True)
    for what, (out, want) in under_vmap("cuda").items():
        # torch's quotient by a number is a product with its inverse on a GPU: a rounding more
        assert (out == want).all() or ((out - want).abs() <= 2.0 ** -22 * want.abs()).all(), what


@pytest.mark.parametrize("V", [37, 5000, 128256])
def test_tokens_not_in_use_among_others(V):
    """Rows of tokens not in use have the biases alone, wherever they are in a tree,
    and the rows around them what their own paths have seen."""
    print(f"\n[case] not in use among others V={V}", flush=True)
    r, g = random.Random(V), torch.Generator().manual_seed(V)
    every = [-1 if i == 0 else max(0, i - 2) if i % 2 == 0 else -2 for i in range(40)]
    trees = [every, [-2] * 9 + [-1, 9, -2, 10], [-2, -1, -2, -2, 1], [-2] * 3, None, random_tree(r, 70, 0.5), [-2, -1], [-1, -2],
             [-1] + [0 if i % 3 else -2 for i in range(1, 600)], random_tree(r, 5, 0.4)]
    new = [40, 13, 5, 3, 6, 70, 2, 2, 600, 5]
    lens, rows = [3000, 70, 64, 40, 90, 700, 66, 30, 700, 3], [0, 1, 2, 3, 4, 5, 5, 5, 6, 7]  # the last: shorter than its tree
    tokens = torch.randint(0, min(V, 300), (8, 3000), generator=g, dtype=torch.int32)
    for some in (slice(0, 10), slice(0, 3), slice(5, 8), slice(8, 10)):
        plan = PagedPlan(lens[some], heads=4, kv_heads=2, new_tokens=new[some], rows=rows[some], parents=trees[some], device="cpu")
        ids = torch.randint(0, V, (8, 7), generator=g, dtype=torch.int32)
        same(torch.randn(plan.tokens, V, generator=g), tokens, plan,
             dict(repetition=1.2, frequency=torch.rand(8, generator=g), presence=0.25, bias=(ids, torch.randn(8, 7, generator=g)),
                  prompts=torch.arange(8, dtype=torch.int32) * 30))
