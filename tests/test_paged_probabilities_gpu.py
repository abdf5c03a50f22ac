"""How the attention over pages holds its probabilities, against float64
formulas where their 16-bit form can lose something.

Every case prints its name before touching the GPU.
"""
import pytest
import torch

from santa_amd.paged import PagedPlan, paged_attention

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("top", [0.0, 1000.0])
@pytest.mark.parametrize("GH, new", [(8, 1), (40, 1), (256, 1), (128, 2)])
def test_many_small_probabilities(GH, new, top):
    """One token of weight 1 and 131 thousand of about 2^-25 each, which f16 does
    not hold: together they make up the output, since the first one's value is 0.
    All of a sequence's tokens are one workgroup's, so that they share the first
    one's reference.  top: the first token's score (1000: subtracted before it is
    scaled)."""
    n, D, page, KVH, B = 131072 + 37, 64, 64, 32, 16
    print(f"\n[case] small probabilities GH={GH} new={new} top={top}", flush=True)
    g = torch.Generator().manual_seed(GH + new)
    k, v = torch.zeros(n, D), torch.rand(n, D, generator=g) + 0.5
    steps = torch.tensor([-17.0, -17.5, -18.0])  # f16 numbers behind 1000, too
    k[:, 0] = top + steps[torch.randint(0, 3, (n,), generator=g)]
    k[5, 0], v[5] = top, 0.0
    pages = -(-n // page)
    pools = []
    order = torch.randperm(pages, generator=g)
    for x in (k, v):
        x = torch.cat([x, torch.full((pages * page - n, D), float("nan"))]).to("cuda", F16)
        pool = torch.empty(pages, page, 1, D, dtype=F16, device="cuda")
        pool[order.cuda()] = x.view(pages, page, 1, D)
        pools.append(pool.expand(-1, -1, KVH, -1))
    q = torch.zeros(B * new, KVH * GH, D, device="cuda", dtype=F16)
    q[..., 0] = 1.0
    plan = PagedPlan([n] * B, heads=KVH * GH, kv_heads=KVH, new_tokens=new, rows=[0] * B)
    items = plan._data[:16 * plan._info.items].view(-1, 16).cpu()
    assert (items[:, 3] - items[:, 2]).max() > n - new - 1
    out = paged_attention(q, *pools, order.int().cuda()[None], plan, scale=1.0).double().cpu().view(B, new, -1, D)
    for i in range(new):
        m = n - new + i + 1
        p = (k[:m, 0].double() - top).exp()
        vh = v[:m].to(F16).double()
        want = (p @ vh) / p.sum()
        # the output's rounding; half of the smallest f16 number, 2^-25, for every probability, relative to a largest
        # of 2^7 or more, on sum and mass; and, of the mean, a rounding of every probability that is a normal number,
        # the float32 exponentials' (exponents up to 2^11 of 24 bits) and the sums'
        bound = 2.0 ** -11 * want + m * 2.0 ** -32 * (1.5 + want) + (2.0 ** -11 + 2.0 ** -12) * want + 2.0 ** -25
        err = (out[:, i] - want).abs()
        assert (err <= bound).all(), (err / bound).max().item()
