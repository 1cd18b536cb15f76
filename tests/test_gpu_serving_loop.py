"""The serving loop in states that a program can bring it into."""

import pytest
import torch

from tinygrad_mi355x.decoder import random_weights
from tinygrad_mi355x.serving import ServingDecoder
from test_gpu_serving_decoder import SMALL, prompts_of

pytestmark = pytest.mark.gpu


def test_prompts_need_the_prefix(dev):
    """Pages of a prefix that was never run through the model are not attended to."""
    d = ServingDecoder(random_weights(SMALL, dev, seed=20), SMALL, 2, 192, 16, prefix=64)
    u = torch.rand((2, 3), device=dev)
    for call in (lambda: d.prefill(prompts_of(dev, 2, 4)), lambda: d.generate(prompts_of(dev, 2, 4), 3, u)):
        with pytest.raises(RuntimeError, match="load_prefix"):
            call()
    with pytest.raises(ValueError):
        d.load_prefix(prompts_of(dev, 1, 64)[0] + SMALL.vocab)
    with pytest.raises(RuntimeError, match="load_prefix"):
        d.prefill(prompts_of(dev, 2, 4))
    d.load_prefix(prompts_of(dev, 1, 64)[0])
    first = d.generate(prompts_of(dev, 2, 4), 3, u)
    assert torch.equal(d.generate(prompts_of(dev, 2, 4), 3, u), first)  # loaded once
