"""The checked steps of tests/test_verified_steps.py on the GPU.  Every case prints its
name before touching the GPU."""
import pytest
import torch

from test_verified_steps import checked_steps

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_steps(dtype):
    print(f"\n[case] checked steps {dtype}", flush=True)
    shares = checked_steps(dtype, "cuda")
    assert len(shares) > 150 and max(shares) <= 1
