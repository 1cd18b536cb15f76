"""Refusals of the mixture-of-experts operators: no GPU needed."""

import pytest
import torch

from tinygrad_mi355x.experts import route
from tinygrad_mi355x.runtime import kernels as K


# ----------------------------------------------------------------------------- routing
@pytest.mark.parametrize("logits,kw", [
    (torch.zeros(8), {}), (torch.zeros(4, 8, 2), {}), (torch.zeros(4, 8, dtype=torch.float64), {}), (torch.zeros(4, 0), {}),
    (torch.zeros(2, 1025), {}), (torch.zeros(8, 4).t(), {}), (torch.zeros(1, 8).expand(4, 8), {}),
    (torch.zeros(4, 8), dict(top_k=0)), (torch.zeros(4, 8), dict(top_k=9)), (torch.zeros(4, 8), dict(top_k=2.0)),
    (torch.zeros(4, 8), dict(score="relu")), (torch.zeros(4, 8), dict(groups=3)), (torch.zeros(4, 8), dict(groups=0)),
    (torch.zeros(4, 130), dict(groups=65)), (torch.zeros(4, 8), dict(groups=4, top_groups=5)),
    (torch.zeros(4, 8), dict(groups=4, top_groups=0)), (torch.zeros(4, 8), dict(groups=4, top_groups=1, top_k=3)),
    (torch.zeros(4, 8), dict(scale=float("inf"))), (torch.zeros(4, 8), dict(bias=torch.zeros(7))),
    (torch.zeros(4, 8), dict(bias=torch.zeros(8, dtype=torch.bfloat16))), (torch.zeros(4, 8), dict(bias=torch.zeros(16)[::2])),
    (torch.zeros(4, 8), dict(bias=torch.zeros(8, device="meta")))])
def test_route_refuses(logits, kw):
    with pytest.raises(ValueError):
        route(logits, kw.pop("top_k", 2), **kw)


def test_route_needs_the_device():
    with pytest.raises(RuntimeError):
        route(torch.zeros(4, 8), 2)


@pytest.mark.parametrize("args", [
    (9, 4, 8, 8, None, 0, 1, 1, 2, 1, 1.0), (13, -1, 8, 8, None, 0, 1, 1, 2, 1, 1.0), (13, 4, 1025, 1025, None, 0, 1, 1, 2, 1, 1.0),
    (13, 4, 8, 7, None, 0, 1, 1, 2, 1, 1.0), (13, 4, 8, 8, None, 2, 1, 1, 2, 1, 1.0), (13, 4, 8, 8, None, 0, 3, 1, 2, 1, 1.0),
    (13, 4, 8, 8, None, 0, 2, 3, 2, 1, 1.0), (13, 4, 8, 8, None, 0, 2, 1, 5, 1, 1.0), (13, 4, 8, 8, None, 0, 1, 1, 0, 1, 1.0),
    (13, 4, 8, 8, None, 0, 1, 1, 2, 1, float("nan")), (13, 4, 8, 8, None, 0, 1, 1, 2, 1, 1.0)])
def test_route_entry_point_refuses(args):
    """What the C entry point is given is checked before any launch; the last one has no operands."""
    with pytest.raises(ValueError):
        K.call("tgm_route", None, *args, None, None, None)
