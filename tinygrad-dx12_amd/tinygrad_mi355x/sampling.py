"""Token sampling from logits with given random numbers (include/tgm_serving.h).

The reference has no model code; this serves models around its packed matmul
(alexandreteles/tinygrad-dx12 src/tinygrad_dx12/codegen/decomp/dx12.py:108-112).
"""

from __future__ import annotations

import torch

from tinygrad_mi355x.rotary import _DT
from tinygrad_mi355x.runtime import kernels as K

MAX_VOCAB = 1 << 20
_workspace_of: dict[tuple, int] = {}


def _per_row(value, name: str, rows: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if isinstance(value, torch.Tensor):
        if value.dtype is not dtype or value.dim() != 1 or value.shape[0] != rows or not value.is_contiguous():
            raise ValueError(f"{name} must be a number or contiguous {dtype} [{rows}], got {value.dtype} {tuple(value.shape)}")
        if value.device != device:
            raise ValueError(f"{name} is on {value.device}, not on {device}")
        return value
    return torch.full((rows,), value, dtype=dtype, device=device)


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
    if logits.dim() != 2 or logits.dtype not in _DT:
        raise ValueError(f"logits must be float32, float16 or bfloat16 [rows, vocab], got {logits.dtype} "
                         f"{tuple(logits.shape)}")
    rows, vocab = logits.shape
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"the vocabulary must hold 1 to {MAX_VOCAB} tokens, got {vocab}")
    if vocab > 1 and logits.stride(1) != 1 or rows > 1 and logits.stride(0) < vocab:
        raise ValueError("rows of logits must be contiguous and apart")
    device = logits.device
    u = _per_row(u, "u", rows, torch.float32, device)
    temperature = _per_row(temperature, "temperature", rows, torch.float32, device)
    if top_k is not None:
        top_k = _per_row(top_k, "top_k", rows, torch.int32, device)
    if top_p is not None:
        top_p = _per_row(top_p, "top_p", rows, torch.float32, device)
    if min_p is not None:
        min_p = _per_row(min_p, "min_p", rows, torch.float32, device)
    if out is not None:
        _per_row(out, "out", rows, torch.int32, device)
    K.require_device(logits)
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=device)
    dt = _DT[logits.dtype]
    key = (rows, vocab, dt)
    need = _workspace_of.get(key)
    if need is None:
        need = _workspace_of[key] = K.load_library().tgm_sample_workspace(*key)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    K.call("tgm_sample", logits.data_ptr(), dt, rows, vocab, max(logits.stride(0), vocab), u.data_ptr(),
           temperature.data_ptr(), K.ptr(top_k), K.ptr(top_p), K.ptr(min_p), out.data_ptr(), K.ptr(workspace), need,
           K.stream_of(logits))
    return out
