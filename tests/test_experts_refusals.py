"""Refusals of the mixture-of-experts operators at the ends of their arguments: no GPU needed."""

import pytest
import torch

from test_experts_host import experts_arg
from tinygrad_mi355x.experts import route
from tinygrad_mi355x.runtime import kernels as K


@pytest.mark.parametrize("kw", [dict(scale=torch.tensor(2.0)), dict(scale=1e39), dict(scale=-1e39), dict(scale=10 ** 400), dict(scale=float("nan")),
                                dict(scale=None), dict(scale="2"), dict(renormalize=torch.tensor(True))])
def test_route_refuses_what_is_no_number(kw):
    """A tensor's value could change between calls that look alike; a scale beyond 32 bits would be infinite."""
    with pytest.raises(ValueError):
        route(torch.zeros(4, 8), 2, **kw)


@pytest.mark.parametrize("scale", [1e39, -1e39])
def test_route_entry_point_refuses_scales(scale):
    with pytest.raises(ValueError, match="scale"):
        K.call("tgm_route", 4096, 13, 4, 8, 8, None, 0, 1, 1, 2, 1, scale, 4096, 4096, None)


@pytest.mark.parametrize("tokens,ldx,ldy", [(3, 1 << 61, 256), (5, 1 << 60, 256), (3, 1 << 62, 256), (3, 256, 1 << 62), (4, 256, 1 << 61)])
def test_experts_rows_whose_distance_passes_64_bits(tokens, ldx, ldy):
    """They are refused before anything is computed from the products, which wrap to small numbers."""
    with pytest.raises(ValueError):
        K.call("tgm_experts_apply", experts_arg(), 4096, 12, tokens, ldx, 4096, 4096, 2, 4096, 12, ldy, 4096, 1 << 40, None)


@pytest.mark.parametrize("ld", [1 << 61, 1 << 62])
def test_logits_rows_whose_distance_passes_64_bits(ld):
    with pytest.raises(ValueError):
        K.call("tgm_route", 4096, 13, 5, 8, ld, None, 0, 1, 1, 2, 1, 1.0, 4096, 4096, None)
    with pytest.raises(ValueError):
        K.call("tgm_log_probs", 4096, 13, 5, 8, ld, 4096, 2, 4096, 4096, 4096, 4096, 4096, None, 0, None)
