"""How the attention over pages holds its probabilities, against float64
formulas where their 16-bit form can lose something.

Every case prints its name before touching the GPU.
"""
import math

import pytest
import torch

from santa_amd.paged import PagedPlan, paged_attention
from santa_amd.runtime import ExactDecodeBackend
from test_shared_pages_gpu import _case, _check, _reference

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


# rows of a pass over the same tokens, in one block, two, and behind prefixes: lens, prefixes, H, KVH, D, page, type
DECODES = [
    ([500, 20], [], 17, 1, 128, 16, BF), ([500, 400], [], 40, 1, 64, 16, F16), ([300], [], 128, 1, 128, 16, BF),
    ([300, 700], [], 256, 1, 64, 8, BF), ([2000] * 40, [(list(range(40)), 1984)], 32, 8, 128, 16, BF),
    ([513 + i for i in range(70)], [(list(range(70)), 512)], 8, 4, 64, 64, F16),
    ([900 + i for i in range(9)], [(list(range(9)), 832)], 16, 4, 128, 32, F16),
    ([400, 390, 380, 10, 399], [([2, 0, 4], 320)], 24, 2, 128, 32, BF),
]


def _tight(out, q, k, v, table, lens, new):
    """Probabilities in two parts: the second one, at most two steps of the first,
    is rounded (4 eps^2 of the mean of |v|), or is less than half of the smallest
    number, 2^-25 of a reference of 2^7, in f16."""
    want, mean, off = _reference(q, k, v, table, lens, new)
    eps = torch.finfo(q.dtype).eps / 2
    bound = eps * want.abs() + (4 * eps * eps + off) * (1 + eps) * mean
    if q.dtype == F16:
        bound += 2.0 ** -25 + 2 * max(lens) * 2.0 ** -32 * v.nan_to_num(0.0).abs().max()
    return ((out.double() - want).abs() / bound).max().item()


@pytest.mark.parametrize("case", range(len(DECODES)))
def test_decode_steps_are_not_rounded(case):
    """A batch of single tokens has the values of float32 probabilities, whatever
    number of rows reads the same tokens; asked for, they are rounded."""
    lens, prefixes, H, KVH, D, page, dtype = DECODES[case]
    print(f"\n[case] decode step {case} lens={lens[:6]} H={H} KVH={KVH} D={D} page={page} {dtype}", flush=True)
    new = [1] * len(lens)
    q, k, v, table, plan = _case(lens, new, prefixes, H, KVH, D, page, dtype, case)
    out = paged_attention(q, k, v, table, plan)
    assert torch.isfinite(out).all() and _tight(out, q, k, v, table, lens, new) <= 1
    assert torch.equal(out, paged_attention(q, k, v, table, plan, rounded=False))
    less = paged_attention(q, k, v, table, plan, rounded=True)
    _check(less, _reference(q, k, v, table, lens, new), dtype)
    assert not torch.equal(less, out)  # a rounded form may lie within the bound of the other, but is not the same


@pytest.mark.parametrize("lens, new, prefixes, H, KVH, D, dtype, rounds", [
    ([300, 90], [8, 5], [], 4, 1, 128, BF, False), ([300, 90], [9, 5], [], 4, 1, 64, F16, True),
    ([700, 650, 300, 66], [90, 1, 0, 2], [([0, 1, 2, 3], 64)], 7, 1, 128, BF, True),
    ([900, 850], [260, 300], [([0, 1], 512)], 8, 2, 128, F16, True), ([130, 64], [130, 64], [], 8, 2, 64, BF, True),
    ([200] * 9, [4] * 9, [(list(range(9)), 128)], 8, 1, 128, F16, False)])
def test_several_tokens_round_where_asked(lens, new, prefixes, H, KVH, D, dtype, rounds):
    """Several new tokens: rounded from more than 32 rows on, unless the caller
    asks for the other; masked tokens in either form."""
    print(f"\n[case] several tokens lens={lens[:4]} new={new[:4]} H={H} D={D} {dtype}", flush=True)
    q, k, v, table, plan = _case(lens, new, prefixes, H, KVH, D, 8, dtype, 3)
    out = [paged_attention(q, k, v, table, plan, rounded=r) for r in (False, True, None)]
    assert torch.equal(out[2], out[rounds]) and plan._info.rounded == rounds
    assert _tight(out[0], q, k, v, table, lens, new) <= 1
    _check(out[1], _reference(q, k, v, table, lens, new), dtype)


@pytest.mark.parametrize("H, D, dtype", [(17, 128, BF), (40, 64, BF), (128, 128, F16), (256, 64, F16), (256, 128, BF)])
def test_infinite_values_in_two_parts(H, D, dtype):
    """An infinite value of a token that a row attends to gives an infinity of its
    sign in its dim, whatever the second part of its probability is, and other
    dims stay as they are."""
    print(f"\n[case] infinite values in two parts H={H} D={D} {dtype}", flush=True)
    lens, new = [300, 70], [2, 1]
    q, k, v, table, plan = _case(lens, new, [], H, 1, D, 8, dtype, 5)
    q.mul_(0.05)  # every token counts: probabilities above 2^-10 of the largest
    clean = paged_attention(q, k, v, table, plan, rounded=False)
    for b, n, d, x in ((0, 3, 1, math.inf), (0, 130, 2, -math.inf), (0, 131, 2, -math.inf), (0, 299, 3, math.inf),
                       (1, 0, 4, -math.inf), (1, 69, 5, math.inf)):
        v[table[b, n // 8].long(), n % 8, 0, d] = x
    want = clean.clone()
    want[:2, :, 1], want[:2, :, 2], want[1, :, 3] = math.inf, -math.inf, math.inf
    want[2, :, 4], want[2, :, 5] = -math.inf, math.inf
    assert torch.equal(paged_attention(q, k, v, table, plan, rounded=False), want)


def test_exact_backend():
    """ExactDecodeBackend.decode_paged: lengths on the GPU, a plan for all layers,
    the values of float32 probabilities for any number of query heads, and a
    captured step."""
    print("\n[case] the exact backend over pages", flush=True)
    lens, shared = [700, 300, 650], [([0, 2], 640)]
    q, k, v, table, plan = _case(lens, [1] * 3, shared, 40, 1, 128, 16, BF, 2)
    backend = ExactDecodeBackend()
    alone = backend.decode_paged(q, k, v, table, lens)
    assert _tight(alone, q, k, v, table, lens, [1] * 3) <= 1
    for x in (torch.tensor(lens), torch.tensor(lens, device="cuda"), torch.tensor(lens, device="cuda").int()):
        assert torch.equal(backend.decode_paged(q, k, v, table, x), alone)
    together = backend.decode_paged(q, k, v, table, plan)
    assert _tight(together, q, k, v, table, lens, [1] * 3) <= 1
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [backend.decode_paged(q, k, v, table, plan) for _ in range(2)]
    for _ in range(3):
        q.normal_()
        graph.replay()
        want = backend.decode_paged(q, k, v, table, plan)
        assert torch.equal(out[0], want) and torch.equal(out[1], want)
