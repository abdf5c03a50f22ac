"""Tensors on different devices are refused, those without a number among them (CPU
and meta)."""
import pytest
import torch

from santa_amd.logits import adjust_logits
from santa_amd.paged import PagedPlan, paged_attention, rope_append


def test_paged_calls():
    lens = [20, 9]
    plan = PagedPlan(lens, heads=4, kv_heads=2, device="cpu")
    q, qkv, cos = torch.randn(2, 4, 16), torch.randn(2, 8, 16), torch.randn(2, 16)
    k, v, norm = torch.randn(6, 8, 2, 16), torch.randn(6, 8, 2, 16), torch.ones(16)
    table = torch.arange(6, dtype=torch.int32).view(2, 3)
    paged_attention(q, k, v, table, plan)
    rope_append(qkv, cos, cos, k, v, table, plan, q_norm=norm, k_norm=norm)
    for name in "kvt":
        args = [x.to("meta") if n == name else x for n, x in zip("kvt", (k, v, table))]
        with pytest.raises(ValueError, match="device mismatch"):
            paged_attention(q, *args, plan)
        with pytest.raises(ValueError, match="device mismatch"):
            rope_append(qkv, cos, cos, *args, plan)
    for args, kw in (((cos.to("meta"), cos), {}), ((cos, cos.to("meta")), {}), ((cos, cos), {"q_norm": norm.to("meta")}),
                     ((cos, cos), {"k_norm": norm.to("meta")})):
        with pytest.raises(ValueError, match="must have the device"):
            rope_append(qkv, *args, k, v, table, plan, **kw)
    with pytest.raises(ValueError):
        paged_attention(q.to("meta"), k, v, table, plan)


def test_rules():
    x, tokens = torch.randn(2, 40), torch.zeros(2, 9, dtype=torch.int32)
    ids, values = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    meta = {"prompts": torch.zeros(2, dtype=torch.int32), "repetition": torch.ones(2), "frequency": torch.ones(2),
            "presence": torch.ones(2), "allowed": torch.zeros(2, 2, dtype=torch.int32)}
    adjust_logits(x, tokens, [9, 4], bias=(ids, values), **meta)
    for name, t in meta.items():
        with pytest.raises(ValueError, match=name):
            adjust_logits(x, tokens, [9, 4], **{name: t.to("meta")})
    for bias in ((ids.to("meta"), values), (ids, values.to("meta"))):
        with pytest.raises(ValueError, match="bias"):
            adjust_logits(x, bias=bias)
    with pytest.raises(ValueError, match="tokens"):
        adjust_logits(x, tokens.to("meta"), [9, 4])
