"""Rules on logits, on the CPU, at the edges of what a call may say."""
import pytest
import torch

from santa_amd.logits import adjust_logits


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
