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

import numbers
import struct
from typing import NamedTuple

import torch

from tinygrad_mi355x.codegen.decomp.mi355x import MX_FORMATS, PackedTensor
from tinygrad_mi355x.rotary import _DT, Plans
from tinygrad_mi355x.runtime import kernels as K
from tinygrad_mi355x.runtime.overlap import Apart

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

    NaN ranks behind everything and counts as -infinity in a group's sum; a row with a NaN, or with +infinity under a softmax,
    has NaN weights (and softmax scores of NaN); chosen logits that are all -infinity have weights of zero.
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
    # plans are looked up by the values of both, which a tensor would change behind its place in the look-up
    if not isinstance(scale, numbers.Real) or not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"scale must be a finite number of 32 bits, got {scale!r}")
    if isinstance(renormalize, torch.Tensor):
        raise ValueError("renormalize must be a truth value, not a tensor")
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.shape != (experts,) or not bias.is_contiguous():
            raise ValueError(f"bias must be contiguous float32 [{experts}], got {bias.dtype} {tuple(bias.shape)}")
        if bias.device != logits.device:
            raise ValueError(f"bias is on {bias.device}, not on {logits.device}")
    K.require_device(logits)
    head = (_DT[logits.dtype], tokens, experts, max(logits.stride(0), experts))
    return _plans.keep(sig, ((SCORES[score], groups, top_groups, top_k, bool(renormalize), float(scale)), head,
                             (tokens, top_k), logits.get_device()))


class PackedExperts:
    """The feed-forward blocks of a layer's experts on packed weights: gate_up [experts, 2 ffn, hidden], gate (2 i) and up
    (2 i + 1) rows in turn as in ``DecoderWeights``, and down [experts, hidden, ffn].

    Both of one format, hidden and ffn multiples of 128: fp4_e2m1, fp6_e2m3 or fp6_e3m2 with E8M0 scales per 32 values (or
    none) for bfloat16 activations; int4 or uint4 with float16, bfloat16 or float32 scales per 32, 64 or 128 (or none) for
    float16 ones.
    """

    def __init__(self, gate_up: PackedTensor, down: PackedTensor) -> None:
        for w, name in ((gate_up, "gate_up"), (down, "down")):
            if not isinstance(w, PackedTensor) or len(w.shape) != 3:
                raise ValueError(f"{name} must be a PackedTensor [experts, rows, columns]")
        self.experts, rows, self.hidden = gate_up.shape
        self.ffn = rows // 2
        if rows % 2 or down.shape != (self.experts, self.hidden, self.ffn):
            raise ValueError(f"down must be [{self.experts}, {self.hidden}, {rows / 2:g}] beside gate_up {gate_up.shape}, got {down.shape}")
        if not 1 <= self.experts <= MAX_EXPERTS:
            raise ValueError(f"a layer holds 1 to {MAX_EXPERTS} experts, got {self.experts}")
        if not self.hidden or not self.ffn or self.hidden % 128 or self.ffn % 128:
            raise ValueError(f"hidden and ffn must be multiples of 128, got {self.hidden} and {self.ffn}")
        if gate_up.format != down.format or _scales(gate_up) != _scales(down) or gate_up.device != down.device:
            raise ValueError("gate_up and down must be of one format, with scales of one type and block, on one device")
        integer = gate_up.format not in MX_FORMATS
        if gate_up.scales is not None:
            dt, block = _scales(gate_up)
            if integer and (dt not in _DT or block not in (32, 64, 128)):
                raise ValueError(f"{gate_up.format} experts take float16, bfloat16 or float32 scales per 32, 64 or 128 values, got "
                                 f"{dt} per {block}")
            if not integer and (dt is not torch.float8_e8m0fnu or block != 32):
                raise ValueError(f"{gate_up.format} experts take E8M0 scales per 32 values, got {dt} per {block}")
        for w, name in ((gate_up, "gate_up"), (down, "down")):
            if not w.data.is_contiguous() or w.scales is not None and not w.scales.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if w.data.data_ptr() % 16 or w.scales is not None and w.scales.data_ptr() % 4:
                raise ValueError(f"codes of {name} must be 16-byte and scales 4-byte aligned")
        self.gate_up, self.down, self.device = gate_up, down, gate_up.device
        self.dtype = torch.float16 if integer else torch.bfloat16  # of the activations
        dt, block = _scales(gate_up)
        # struct tgm_experts; the weights are never replaced
        self.arg = struct.pack("PPPPqqqqqq", gate_up.data.data_ptr(), K.ptr(gate_up.scales) or 0, down.data.data_ptr(),
                                K.ptr(down.scales) or 0, self.experts, self.hidden, self.ffn, K.FORMAT_IDS[gate_up.format],
                                -1 if dt is None else K.dtype_id(dt), block)
        self._plans = Plans()

    def apply(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
        """The weighted sum of each token's experts: x [tokens, hidden] of ``dtype``, ids (int32) and weights (float32)
        [tokens, top_k] as ``route`` gives them.

        ``out`` [tokens, hidden] is of x's type or float32 (x's type), with contiguous rows; it may be x, and shares no memory
        with weights.  An id outside 0 .. experts - 1 names no expert and adds nothing, whatever its weight: a row without any
        is zero.  The same expert may be named twice.  Products and sums are float32; silu(gate) * up is rounded to x's type
        before the down product.
        x starts at a multiple of 16 bytes, and its rows lie a multiple of 8 values apart.
        """
        sig = (x.shape, x.stride(), x.dtype, x.get_device(), ids.shape, ids.stride(), ids.dtype, ids.get_device(), weights.shape,
               weights.stride(), weights.dtype, weights.get_device())
        if out is not None:
            sig += (out.shape, out.stride(), out.dtype, out.get_device())
        plan = self._plans.get(sig)
        if plan is None:
            plan = self._apply_plan(sig, x, ids, weights, out)
        head, top_k, tail, need, index, apart = plan
        if out is None:
            out = x.new_empty(x.shape)
        else:
            apart.check(out, weights, "weights")  # which are read while it is written
        if x.shape[0]:
            # the workspace is of the caching allocator, so that calls on several streams never share one; held until the
            # launches, or another thread's call on this stream could be given its memory before them
            workspace = x.new_empty(need, dtype=torch.uint8)
            K.call("tgm_experts_apply", self.arg, x.data_ptr(), *head, ids.data_ptr(), weights.data_ptr(), top_k,
                   out.data_ptr(), *tail, workspace.data_ptr(), need, K.stream_on(index))
        return out

    def workspace_bytes(self, tokens: int, top_k: int) -> int:
        """The workspace that a call on so many tokens takes, which one on fewer can take too."""
        return K.load_library().tgm_experts_workspace(self.arg, tokens, top_k)

    def _apply_plan(self, sig, x, ids, weights, out) -> tuple:
        _check_rows(x, "x", self.hidden)
        if x.dtype is not self.dtype:
            raise ValueError(f"x must be {self.dtype} beside {self.gate_up.format} experts, got {x.dtype}")
        tokens = x.shape[0]
        if ids.dtype is not torch.int32 or ids.dim() != 2 or ids.shape[0] != tokens or ids.shape[1] < 1 or not ids.is_contiguous():
            raise ValueError(f"ids must be contiguous int32 [{tokens}, top_k], got {ids.dtype} {tuple(ids.shape)}")
        if weights.dtype is not torch.float32 or weights.shape != ids.shape or not weights.is_contiguous():
            raise ValueError(f"weights must be contiguous float32 {tuple(ids.shape)}, got {weights.dtype} {tuple(weights.shape)}")
        ldy, odt = self.hidden, x.dtype
        if out is not None:
            _check_rows(out, "out", self.hidden)
            if out.shape != x.shape or out.dtype not in (x.dtype, torch.float32):
                raise ValueError(f"out must be {x.dtype} or float32 {tuple(x.shape)}, got {out.dtype} {tuple(out.shape)}")
            ldy, odt = max(out.stride(0), self.hidden), out.dtype
        for t, name in ((x, "x"), (ids, "ids"), (weights, "weights"), (out, "out")):
            if t is not None and t.device != self.device:
                raise ValueError(f"{name} is on {t.device}, the experts on {self.device}")
        ldx = max(x.stride(0), self.hidden)
        if ldx % 8 and tokens > 1:
            raise ValueError(f"rows of x must be 16-byte aligned, got a stride of {ldx}")
        K.require_device(x)
        need = self.workspace_bytes(tokens, ids.shape[1])
        return self._plans.keep(sig, ((_DT[x.dtype], tokens, ldx), ids.shape[1], (_DT[odt], ldy), need, x.get_device(),
                                       None if out is None else Apart(out, weights)))


def _scales(w: PackedTensor) -> tuple:
    return (None, 32) if w.scales is None else (w.scales.dtype, w.block_size)


def _check_rows(t: torch.Tensor, name: str, hidden: int) -> None:
    if t.dim() != 2 or t.shape[1] != hidden:
        raise ValueError(f"{name} must be [tokens, {hidden}], got {tuple(t.shape)}")
    if t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < hidden:
        raise ValueError(f"rows of {name} must be contiguous and apart")
