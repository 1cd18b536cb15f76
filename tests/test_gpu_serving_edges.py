"""The serving operators where their arguments end: filters that keep one token, infinite temperatures, queries and scores
that are not finite, positions that nobody wrote, tensors that overlap (tolerances: test_gpu_serving.py)."""

import math

import pytest
import torch

from test_gpu_serving import BF16, F32, check_sample

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- sampling
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [400, 513, 1000, 2048, 5000])
@pytest.mark.parametrize("top_p", [0.0, -1.0, -math.inf])
def test_sample_keeps_the_largest_of_flat_rows(dev, dtype, n, top_p):
    """A top_p of 0 and less keeps the first maximum alone, also among tokens of nearly one weight."""
    print(f"flat rows {dtype} {n} {top_p}", flush=True)
    g = torch.Generator().manual_seed(n)
    flat, spread = torch.rand(2, n, generator=g) * 0.001, torch.randn(2, n, generator=g)
    for x, temperature in ((flat, 1.0), (spread, 500.0), (torch.ones(2, n), 0.7)):
        x = x.to(dtype)
        for u, min_p in ((torch.rand(2, generator=g), 0.0), (torch.zeros(2), 0.0), (torch.rand(2, generator=g), 0.5)):
            got = check_sample(dev, x, u, temperature, 0, top_p, min_p)
            assert torch.equal(got.cpu().long(), x.float().argmax(1))
