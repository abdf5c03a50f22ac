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
@pytest.mark.parametrize("H, new", [(8, 1), (40, 1), (256, 1), (128, 2)])
def test_many_small_probabilities(H, new, top):
    """One token of weight 1 and 131 thousand of about 2^-25 each, which f16 does
    not hold: together they make up the output, since the first one's value is 0.
    top: the first token's score (1000: subtracted before it is scaled)."""
    n, D, page = 131072 + 37, 64, 64
    print(f"\n[case] small probabilities H={H} new={new} top={top}", flush=True)
    g = torch.Generator().manual_seed(H + new)
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
        pools.append(pool)
    q = torch.zeros(new, H, D, device="cuda", dtype=F16)
    q[..., 0] = 1.0
    plan = PagedPlan([n], heads=H, kv_heads=1, new_tokens=new)
    out = paged_attention(q, *pools, order.int().cuda()[None], plan, scale=1.0).double().cpu()
    for i in range(new):
        m = n - new + i + 1
        p = (k[:m, 0].double() - top).exp()
        vh = v[:m].to(F16).double()
        want = (p @ vh) / p.sum()
        # the output's rounding; half of the smallest f16 number, 2^-25, for every probability, relative to a largest
        # of 2^7 or more, on sum and mass; and, of the mean, a rounding of every probability that is a normal number,
        # the float32 exponentials' (exponents up to 2^11 of 24 bits) and the sums'
        bound = 2.0 ** -11 * want + m * 2.0 ** -32 * (1.5 + want) + (2.0 ** -11 + 2.0 ** -12) * want + 2.0 ** -25
        err = (out[i] - want).abs()
        assert (err <= bound).all(), (err / bound).max().item()
