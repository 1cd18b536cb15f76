"""Token sampling from logits with given random numbers (include/tgm_serving.h).

The reference has no model code; this serves models around its packed matmul
(alexandreteles/tinygrad-dx12 src/tinygrad_dx12/codegen/decomp/dx12.py:108-112).
"""

from __future__ import annotations

import torch

from tinygrad_mi355x.rotary import _DT, Plans
from tinygrad_mi355x.runtime import kernels as K

MAX_VOCAB = 1 << 20
_plans = Plans()


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature: torch.Tensor | float = 1.0,
           top_k: torch.Tensor | int | None = None, top_p: torch.Tensor | float | None = None,
           min_p: torch.Tensor | float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row of logits [rows, vocab], int32 [rows].

    Weights are exp((logit - max) / temperature).  top_k keeps the k largest (0: all); top_p keeps the shortest run of
    the largest whose mass reaches its share of what top_k left (1: all; the largest always stays); min_p drops weights
    below its share of the largest.  Equal logits rank by index.  The token is the first kept one whose running sum in
    the vocabulary's order exceeds u times the kept mass: ``u`` float32 [rows] in [0, 1).  A temperature of 0 takes the
    first maximum.  -inf and NaN logits are never taken; a row that holds nothing else gives 0.

    Each parameter is one number, or a contiguous tensor with one per row (float32; top_k int32).
    """
    if out is not None and logits.dim():
        _per_row(out, "out", logits.shape[0], torch.int32, logits.device)
    sig = (logits.shape, logits.stride(), logits.dtype, logits.get_device(), _signature(u), _signature(temperature),
           _signature(top_k), _signature(top_p), _signature(min_p))
    plan = _plans.get(sig)
    if plan is None:
        plan = _plan(sig, logits, u, temperature, top_k, top_p, min_p)
    dt, rows, vocab, ld, need, index, numbers = plan
    if numbers:  # given as plain numbers
        temperature = _filled(temperature, rows, torch.float32, logits.device)
        top_k = _filled(top_k, rows, torch.int32, logits.device)
        top_p = _filled(top_p, rows, torch.float32, logits.device)
        min_p = _filled(min_p, rows, torch.float32, logits.device)
    if out is None:
        out = logits.new_empty(rows, dtype=torch.int32)
    # the workspace is of the caching allocator, so that calls on several streams never share one; held until the launch, or
    # another thread's call on this stream could be given its memory before that
    workspace = logits.new_empty(need, dtype=torch.uint8) if need else None
    if not rows:
        return out
    K.call("tgm_sample", logits.data_ptr(), dt, rows, vocab, ld, u.data_ptr(), temperature.data_ptr(),
           None if top_k is None else top_k.data_ptr(), None if top_p is None else top_p.data_ptr(),
           None if min_p is None else min_p.data_ptr(), out.data_ptr(), K.ptr(workspace), need, K.stream_on(index))
    return out


def _signature(t):
    return (t.shape, t.stride(), t.dtype, t.get_device()) if isinstance(t, torch.Tensor) else type(t)


def _filled(value, rows: int, dtype: torch.dtype, device: torch.device):
    return value if value is None or isinstance(value, torch.Tensor) else torch.full((rows,), value, dtype=dtype, device=device)


def _plan(sig, logits, u, temperature, top_k, top_p, min_p) -> tuple:
    if logits.dim() != 2 or logits.dtype not in _DT:
        raise ValueError(f"logits must be float32, float16 or bfloat16 [rows, vocab], got {logits.dtype} "
                         f"{tuple(logits.shape)}")
    rows, vocab = logits.shape
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"the vocabulary must hold 1 to {MAX_VOCAB} tokens, got {vocab}")
    if vocab > 1 and logits.stride(1) != 1 or rows > 1 and logits.stride(0) < vocab:
        raise ValueError("rows of logits must be contiguous and apart")
    if not isinstance(u, torch.Tensor):
        raise ValueError("u must be a tensor: one random number per row")
    numbers = False
    for value, name, dtype in ((u, "u", torch.float32), (temperature, "temperature", torch.float32),
                               (top_k, "top_k", torch.int32), (top_p, "top_p", torch.float32),
                               (min_p, "min_p", torch.float32)):
        if isinstance(value, torch.Tensor):
            _per_row(value, name, rows, dtype, logits.device)
        elif value is not None:
            if not isinstance(value, (int, float)) or name == "top_k" and not isinstance(value, int):
                raise ValueError(f"{name} must be a number or a tensor, got {value!r}")
            numbers = True
        elif name == "temperature":
            raise ValueError("temperature must be a number or a tensor")
    K.require_device(logits)
    dt = _DT[logits.dtype]
    need = K.load_library().tgm_sample_workspace(rows, vocab, dt)
    return _plans.keep(sig, (dt, rows, vocab, max(logits.stride(0), vocab), need, logits.get_device(), numbers))


def _per_row(t: torch.Tensor, name: str, rows: int, dtype: torch.dtype, device: torch.device) -> None:
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != rows or not t.is_contiguous():
        raise ValueError(f"{name} must be a number or contiguous {dtype} [{rows}], got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
