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


@pytest.mark.parametrize("temperature", [math.inf, 3e38, 1e30])
@pytest.mark.parametrize("n", [300, 1000, 2048, 5000])
def test_sample_at_huge_temperatures(dev, n, temperature):
    """An infinite temperature weighs all finite logits alike; a huge one still tells logits of 3e38 apart."""
    print(f"huge temperature {n} {temperature}", flush=True)
    g = torch.Generator().manual_seed(n)
    for scale in (1.0, 3.3e38):
        x = (torch.rand(3, n, generator=g) * 2 - 1) * scale
        for top_k, top_p, min_p in ((0, 0.9, 0.0), (0, 1.0, 0.5), (n // 2, 0.8, 0.0), (0, 1.0, 0.0)):
            for u in (torch.rand(3, generator=g), torch.zeros(3)):
                check_sample(dev, x, u, temperature, top_k, top_p, min_p)
