"""Float32 rotary tables on the GPU next to the zeros of cos and sin, against float64.

Tolerance: cos and sin are off by at most 16 steps of 2^-24 of themselves (sincospif 4,
a sum, the product with the magnitude, and room for their rounding together); the
angle by 2^-50 of the position (a product, a quotient and a remainder in float64) and,
of what is left of a float32 part of a turn, at most 2 pi 2^-26, by three steps of 2^-24
and its square: 2^-45 with the result's own roundings.

Every case prints its name before touching the GPU.
"""
import pytest
import torch

from santa_amd.paged import RopeScaling, rope_tables
from test_rotary import frequency

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scaling", [None, RopeScaling("llama3", 8.0, 8192), RopeScaling("yarn", 4.0, 4096)])
@pytest.mark.parametrize("dim, interleaved", [(128, False), (64, True), (6, False)])
def test_zeros(dim, interleaved, scaling):
    print(f"\n[case] tables near zeros dim={dim} interleaved={interleaved} {scaling}", flush=True)
    pos = torch.arange(-5, 30000)
    got = rope_tables(pos.cuda(), dim, scaling=scaling, interleaved=interleaved, dtype=torch.float32)
    pairs = [frequency(i, dim, 10000.0, scaling) for i in range(dim // 2)]
    angle = pos.double()[:, None] * torch.tensor([f for f, _ in pairs], dtype=torch.float64)
    angle = angle.repeat_interleave(2, -1) if interleaved else torch.cat([angle, angle], -1)
    want = angle.cos() * pairs[0][1], angle.sin() * pairs[0][1]
    near = 0
    for a, b in zip(got, want):
        bound = 2.0 ** -20 * b.abs() + pos.abs()[:, None] * 2.0 ** -50 + 2.0 ** -45
        assert ((a.double().cpu() - b).abs() <= bound).all()
        near += int(((b.abs() > 1e-6) & (b.abs() < 1e-3)).sum())
    assert near > 100  # where a part of a turn rounded to float32 is off by more than the bound
