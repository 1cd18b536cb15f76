"""Rotary positions of query and key heads (include/tgm_serving.h).

The reference has no model code; this serves models around its packed matmul
(alexandreteles/tinygrad-dx12 src/tinygrad_dx12/codegen/decomp/dx12.py:108-112).

A ``Rotary`` holds what a model's configuration states: which pairs of a head's values rotate, how fast,
and how the frequencies are scaled for contexts beyond the trained length.
"""

from __future__ import annotations

import math
import struct

import torch

from tinygrad_mi355x.runtime import kernels as K
from tinygrad_mi355x.runtime.overlap import OutLayout

LAYOUTS = {"half": 0, "interleaved": 1}
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_DT = {dt: K.dtype_id(dt) for dt in FLOATS}
_HEADS = struct.Struct("qqqqq").pack


def heads_arg(t: torch.Tensor) -> bytes:
    """struct tgm_heads of a tensor [batch, tokens, heads, head_dim]."""
    sb, st, sh, _ = t.stride()
    return _HEADS(sb, st, sh, t.shape[2], _DT[t.dtype])


class Plans(dict):
    """What calls of one signature (shapes, strides, types, devices) have in common: checked once, then looked up, since
    the checks of a call on a few tokens take longer than its kernel.  Bounded: a program has few signatures."""

    def keep(self, key, plan):
        if len(self) >= 512:
            self.clear()
        self[key] = plan
        return plan


def check_heads(t: torch.Tensor, name: str) -> None:
    """A float tensor [batch, tokens, heads, head_dim], the values of a head contiguous."""
    if t.dim() != 4:
        raise ValueError(f"{name} must be [batch, tokens, heads, head_dim], got {tuple(t.shape)}")
    if t.dtype not in _DT:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if t.stride(3) != 1 and t.shape[3] > 1:
        raise ValueError(f"the values of a head of {name} must be contiguous")


def check_index(t: torch.Tensor, name: str, batch: int, like: torch.Tensor) -> None:
    """One contiguous int32 per sequence beside ``like``."""
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != batch or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 [{batch}], got {t.dtype} {tuple(t.shape)}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """Radians per position of each rotated pair (float64), and the gain on the rotated values.

    Pair i turns by base^(-2 i / rotary_dim) a position.  ``scaling`` stretches that for long contexts:

    * ``{"kind": "linear", "factor": f}``: every frequency divided by f;
    * ``{"kind": "ntk", "factor": f}``: the base times f^(n / (n - 2)), n = rotary_dim: the slowest pair slows by f,
      the fastest stays;
    * ``{"kind": "yarn", "factor": f, "trained": length}``: pairs that turn over ``fast`` (32) times in the trained
      length stay, pairs that turn under ``slow`` (1) times are divided by f, a ramp over the pairs between; rotated
      values are multiplied by ``gain`` (0.1 ln f + 1).
    """
    n, gain = rotary_dim, 1.0
    spec = dict(scaling or {})
    kind, factor = spec.pop("kind", None), float(spec.pop("factor", 1.0))
    if kind not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown rotary scaling {kind!r}: linear, ntk or yarn")
    if kind and not factor >= 1.0:
        raise ValueError(f"the rotary scaling factor must be at least 1, got {factor}")
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError(f"the rotary base must be above 1, got {base}")
    if kind == "ntk":
        if n < 4:
            raise ValueError("ntk scaling needs a rotary_dim of 4 and more")
        base = base * factor ** (n / (n - 2))
    pair = torch.arange(n // 2, dtype=torch.float64)
    freq = base ** (-2 * pair / n) if n else pair
    if kind == "linear":
        freq = freq / factor
    elif kind == "yarn":
        if "trained" not in spec:
            raise ValueError("yarn scaling needs the trained length")
        trained, fast, slow = float(spec.pop("trained")), float(spec.pop("fast", 32.0)), float(spec.pop("slow", 1.0))
        if not (trained > 0 and fast > 0 and slow > 0):
            raise ValueError("yarn scaling needs positive trained, fast and slow")
        gain = float(spec.pop("gain", 0.1 * math.log(factor) + 1.0))
        # the pair that turns so many times in the trained length
        at = [n * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (fast, slow)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n - 1)
        slowed = ((pair - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq * (1 - slowed) + freq / factor * slowed
    if spec:
        raise ValueError(f"unknown rotary scaling settings {sorted(spec)}")
    return freq, gain


class Rotary:
    """Rotary positions: the leading ``rotary_dim`` values of every head (all of them by default) rotate in pairs.

    ``layout``: "half" pairs value i with i + rotary_dim / 2, "interleaved" 2 i with 2 i + 1.  ``scaling``: see
    ``frequencies``.
    """

    def __init__(self, head_dim: int, rotary_dim: int | None = None, *, base: float = 10000.0, layout: str = "half",
                 scaling: dict | None = None, device: str | torch.device = "cuda") -> None:
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 1 or not 0 <= rotary_dim <= head_dim or rotary_dim % 2:
            raise ValueError(f"rotary_dim must be even and at most head_dim, got {rotary_dim} of {head_dim}")
        if layout not in LAYOUTS:
            raise ValueError(f"unknown rotary layout {layout!r}: half or interleaved")
        self.head_dim, self.rotary_dim, self.base, self.layout = head_dim, rotary_dim, base, layout
        freq, self.gain = frequencies(rotary_dim, base, scaling)
        self.freq = freq.to(device)
        self._plans = Plans()
        self.arg = struct.pack("Pdqq", self.freq.data_ptr(), self.gain, rotary_dim, LAYOUTS[layout])  # struct tgm_rotary

    def check(self, x: torch.Tensor, head_dim: int) -> None:
        if head_dim != self.head_dim:
            raise ValueError(f"heads of {head_dim} values, but the rotary positions are of {self.head_dim}")
        if x.device != self.freq.device:
            raise ValueError(f"heads on {x.device}, the rotary positions on {self.freq.device}")

    def rotate(self, x: torch.Tensor, start: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """x [batch, tokens, heads, head_dim] rotated; token t of sequence b stands at position start[b] + t.

        ``start``: int32 [batch].  ``out`` is x itself or shares no memory with it.  Angles, sines and products are computed in
        64 bits.
        """
        sig = (x.shape, x.stride(), x.dtype, x.get_device(), start.shape, start.stride(), start.dtype, start.get_device())
        plan = self._plans.get(sig)
        if plan is None:
            plan = self._plan(sig, x, start)
        x_arg, out_arg, shape, batch, tokens, index = plan
        if out is None:
            out = x.new_empty(shape)
        else:
            out_sig = (sig, out.shape, out.stride(), out.dtype, out.get_device())
            out_arg, layout = self._plans.get(out_sig) or self._out_plan(out_sig, x, out)
            layout.check(out, x, "x")
        if batch and tokens:
            K.call("tgm_rotate", self.arg, x_arg, x.data_ptr(), out_arg, out.data_ptr(), start.data_ptr(), batch, tokens,
                   self.head_dim, K.stream_on(index))
        return out

    def _out_plan(self, sig, x: torch.Tensor, out: torch.Tensor) -> tuple:
        check_heads(out, "out")
        if out.shape != x.shape or out.dtype is not x.dtype or out.device != x.device:
            raise ValueError("out must be like x")
        return self._plans.keep(sig, (heads_arg(out), OutLayout(out, x)))

    def _plan(self, sig, x: torch.Tensor, start: torch.Tensor) -> tuple:
        check_heads(x, "x")
        batch, tokens, heads, head_dim = x.shape
        self.check(x, head_dim)
        check_index(start, "start", batch, x)
        K.require_device(x)
        row = heads * head_dim
        out_arg = _HEADS(tokens * row, row, head_dim, heads, _DT[x.dtype])
        return self._plans.keep(sig, (heads_arg(x), out_arg, x.shape, batch, tokens, x.get_device()))
