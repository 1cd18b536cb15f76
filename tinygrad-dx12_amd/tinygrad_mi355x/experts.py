"""Mixture-of-experts layers on packed weights (include/tgm_experts.h).

The reference has no model code; this serves models around its packed matmul
(alexandreteles/tinygrad-dx12 src/tinygrad_dx12/codegen/decomp/dx12.py:108-112).

* ``route`` chooses each token's experts from its router logits, and their weights;
* ``PackedExperts`` holds the packed weights of a layer's experts; ``apply`` runs tokens through those that were chosen for
  them.

Results and workspaces come from torch's caching allocator: to replay calls as a graph, capture them with
``torch.cuda.graph``, which keeps their memory in a pool of its own.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from tinygrad_mi355x.rotary import _DT, Plans
from tinygrad_mi355x.runtime import kernels as K

SCORES = {"softmax": 0, "sigmoid": 1}  # enum tgm_route_score
MAX_EXPERTS, MAX_GROUPS = 1024, 64
_plans = Plans()


class Routing(NamedTuple):
    """What ``route`` returns, each [tokens, top_k]: the experts (int32), the best first, and their weights (float32)."""
    ids: torch.Tensor
    weights: torch.Tensor


def route(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
          top_groups: int | None = None, renormalize: bool = True, scale: float = 1.0) -> Routing:
    """The ``top_k`` experts of each token from its router logits [tokens, experts] (float32, float16 or bfloat16).

    A token's scores are the softmax or the sigmoid of its logits; ``bias`` (float32 [experts]) is added for the choice
    alone.  With ``groups`` of neighbouring experts, a group counts by the sum of its two best, and the choice is among the
    ``top_groups`` best groups (all of them).  Equal ones rank by index; the choice is that of values in 64 bits.  The
    weights are the chosen experts' scores, divided by their sum with ``renormalize``, times ``scale``.

    NaN ranks behind everything; a row with a NaN, or with +infinity under a softmax, has NaN weights; chosen scores that
    are all zero (every logit is -infinity) are weights of zero.
    """
    top_groups = groups if top_groups is None else top_groups
    sig = (logits.shape, logits.stride(), logits.dtype, logits.get_device(), top_k, score, groups, top_groups, renormalize,
           scale, None if bias is None else (bias.shape, bias.stride(), bias.dtype, bias.get_device()))
    plan = _plans.get(sig)
    if plan is None:
        plan = _route_plan(sig, logits, top_k, score, bias, groups, top_groups, renormalize, scale)
    args, head, shape, index = plan
    ids, weights = logits.new_empty(shape, dtype=torch.int32), logits.new_empty(shape, dtype=torch.float32)
    if shape[0]:
        K.call("tgm_route", logits.data_ptr(), *head, None if bias is None else bias.data_ptr(), *args, ids.data_ptr(),
               weights.data_ptr(), K.stream_on(index))
    return Routing(ids, weights)


def _route_plan(sig, logits, top_k, score, bias, groups, top_groups, renormalize, scale) -> tuple:
    if logits.dim() != 2 or logits.dtype not in _DT:
        raise ValueError(f"logits must be float32, float16 or bfloat16 [tokens, experts], got {logits.dtype} "
                         f"{tuple(logits.shape)}")
    tokens, experts = logits.shape
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"a router chooses among 1 to {MAX_EXPERTS} experts, got {experts}")
    if experts > 1 and logits.stride(1) != 1 or tokens > 1 and logits.stride(0) < experts:
        raise ValueError("rows of logits must be contiguous and apart")
    if score not in SCORES:
        raise ValueError(f"unknown score {score!r}: softmax or sigmoid")
    for name, value in (("top_k", top_k), ("groups", groups), ("top_groups", top_groups)):
        if not isinstance(value, int):
            raise ValueError(f"{name} must be a whole number, got {value!r}")
    if not 1 <= groups <= MAX_GROUPS or experts % groups:
        raise ValueError(f"groups must be 1 to {MAX_GROUPS} and divide the {experts} experts, got {groups}")
    if not 1 <= top_groups <= groups:
        raise ValueError(f"top_groups must be 1 to {groups}, got {top_groups}")
    if not 1 <= top_k <= experts // groups * top_groups:
        raise ValueError(f"top_k must be 1 to {experts // groups * top_groups}, the experts of {top_groups} groups, got {top_k}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.shape != (experts,) or not bias.is_contiguous():
            raise ValueError(f"bias must be contiguous float32 [{experts}], got {bias.dtype} {tuple(bias.shape)}")
        if bias.device != logits.device:
            raise ValueError(f"bias is on {bias.device}, not on {logits.device}")
    K.require_device(logits)
    head = (_DT[logits.dtype], tokens, experts, max(logits.stride(0), experts))
    return _plans.keep(sig, ((SCORES[score], groups, top_groups, top_k, bool(renormalize), float(scale)), head,
                             (tokens, top_k), logits.get_device()))
