"""The model over a shared paged cache on the GPU: which calls its kernels take.

Every case prints its name before touching the GPU.
"""
import pytest
import torch
from torch.utils.flop_counter import FlopCounterMode

from santa_amd.runtime import NHDCache, RandomLlama
from test_paged import _model_cache
from test_shared_pages_gpu import SMALL

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _logits(model, toks, n):
    """Each sequence of toks [B, n] prefilled in pages but for its last token, which is a decode step."""
    cache = _model_cache(SMALL, "cuda", BF, num_pages=200, page_size=16, max_len=n)
    seqs = cache.add([0] * len(toks))
    model.extend(toks[:, :n - 1], cache, seqs)
    return model.extend(toks[:, n - 1:n], cache, seqs)


def test_modes_see_every_product():
    """Under a dispatch mode the layers run as torch operations."""
    print("\n[case] a flop counter around extend", flush=True)
    model = RandomLlama(SMALL, seed=11, std=0.05, device="cuda", dtype=BF)
    toks = torch.randint(0, SMALL.vocab, (2, 90), generator=torch.Generator().manual_seed(5)).cuda()
    want = _logits(model, toks, 90)
    with FlopCounterMode(display=False) as counter:
        got = _logits(model, toks, 90)
    weights = sum(w.numel() for L in model.layers for w in L.values() if w.dim() == 2)
    seen = sum(n for op, n in counter.get_flop_counts()["Global"].items() if op is not torch.ops.aten.bmm)
    assert seen == 2 * (2 * 90 * weights + 2 * 2 * model.lm_head.numel())  # the attention's are batched products
    # to the tolerance of the runtime's decode against its prefill
    assert (got - want).abs().max() <= 0.05 * want.abs().max()


@pytest.mark.parametrize("change", ["autocast", "float32 norms", "strided norms"])
def test_what_the_kernels_do_not_take(change):
    """Autocast to another type, and norms that are laid out or typed otherwise,
    run the torch expressions, as the prefill's."""
    print(f"\n[case] extend with {change}", flush=True)
    model = RandomLlama(SMALL, seed=11, std=0.05, device="cuda", dtype=BF)
    toks = torch.randint(0, SMALL.vocab, (2, 90), generator=torch.Generator().manual_seed(5)).cuda()
    want = _logits(model, toks, 90)
    for L in model.layers:
        for name in ("ln1", "ln2"):
            if change == "float32 norms":
                L[name] = L[name].float()
            elif change == "strided norms":
                L[name] = torch.stack([L[name]] * 2, -1)[:, 0]
    assert model._fused_layers_take(model.embed[toks[0]]) == (change == "autocast")
    with torch.autocast("cuda", torch.float16, enabled=change == "autocast"):
        if change != "float32 norms":
            got = _logits(model, toks, 90)
            alone = model.prefill(toks, NHDCache(SMALL, 2, 90, BF, "cuda"))
        else:  # the norms' type is that of the products' input, which the weights do not have
            with pytest.raises(RuntimeError, match="dtype"):
                _logits(model, toks, 90)
            return
    for x in (want, alone):
        assert (got - x).abs().max() <= 0.05 * want.abs().max()
