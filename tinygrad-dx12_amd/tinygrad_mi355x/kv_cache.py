"""A paged key/value cache in 8 or 4 bits, and attention over it (include/tgm_serving.h).

The reference has no model code; this serves models around its packed matmul
(alexandreteles/tinygrad-dx12 src/tinygrad_dx12/codegen/decomp/dx12.py:108-112).

``PackedKVCache`` holds pages of ``page_size`` positions.  Keys and values are stored as fp8_e4m3 or fp4_e2m1 codes
with one power-of-two scale per 32 values of a head, as PackedTensor's MX formats store weights.  A page table
(int32 [batch, columns], owned by the caller) names the pages of each sequence in the order of its positions; entries
past what a sequence uses may hold anything (the kernels check every page number).

* ``append`` rotates new keys (and queries), quantises keys and values and writes them at their positions;
* ``read`` gives positions back in a floating type;
* ``attend`` is grouped-query attention of the newest tokens over everything cached, a few tokens (decode) or a chunk
  of a prompt, with or without a prefix that the whole batch shares.

Results and workspaces come from torch's caching allocator: to replay calls as a graph, capture them with
``torch.cuda.graph``, which keeps their memory in a pool of its own.
"""

from __future__ import annotations

import math
import struct
from typing import NamedTuple

import torch

from tinygrad_mi355x.rotary import _DT, _HEADS, Plans, Rotary, check_heads, check_index, heads_arg
from tinygrad_mi355x.runtime import kernels as K
from tinygrad_mi355x.runtime.overlap import OutLayout

FORMATS = {"fp8_e4m3": (0, 8), "fp4_e2m1": (1, 4)}  # enum tgm_kv_format, bits of a code
BLOCK = 32


class Appended(NamedTuple):
    """What ``append`` returns: the rotated queries, and the new keys and values as the cache holds them (None where
    not asked for)."""
    q: torch.Tensor | None
    k: torch.Tensor | None
    v: torch.Tensor | None


class PackedKVCache:
    """Stores of ``pages`` pages: k_data / v_data uint8 [pages, kv_heads, page_size, head_dim (or half of it)] and
    k_scales / v_scales uint8 [pages, kv_heads, head_dim / 32, page_size] (exponent plus 127)."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64, k_format: str = "fp8_e4m3",
                 v_format: str = "fp8_e4m3", device: str | torch.device = "cuda") -> None:
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if pages < 1 or kv_heads < 1:
            raise ValueError("a cache needs at least one page and one head")
        for name, fmt in (("k_format", k_format), ("v_format", v_format)):
            if fmt not in FORMATS:
                raise ValueError(f"unknown {name} {fmt!r}: fp8_e4m3 or fp4_e2m1")
        self.pages, self.kv_heads, self.head_dim, self.page_size = pages, kv_heads, head_dim, page_size
        self.k_format, self.v_format = k_format, v_format
        u8 = dict(dtype=torch.uint8, device=device)
        self.k_data = torch.zeros((pages, kv_heads, page_size, head_dim * FORMATS[k_format][1] // 8), **u8)
        self.v_data = torch.zeros((pages, kv_heads, page_size, head_dim * FORMATS[v_format][1] // 8), **u8)
        self.k_scales = torch.zeros((pages, kv_heads, head_dim // BLOCK, page_size), **u8)
        self.v_scales = torch.zeros((pages, kv_heads, head_dim // BLOCK, page_size), **u8)
        self.device = self.k_data.device
        # struct tgm_kv_cache; the stores are never replaced
        self._arg = struct.pack("PPPPqqqqqq", self.k_data.data_ptr(), self.k_scales.data_ptr(), self.v_data.data_ptr(),
                                self.v_scales.data_ptr(), pages, kv_heads, head_dim, page_size, FORMATS[k_format][0],
                                FORMATS[v_format][0])
        self._scale = 1.0 / math.sqrt(head_dim)
        self._plans = Plans()

    def nbytes(self) -> int:
        return sum(t.numel() for t in (self.k_data, self.k_scales, self.v_data, self.v_scales))

    def _check_table(self, table: torch.Tensor, batch: int) -> None:
        if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != batch:
            raise ValueError(f"the page table must be int32 [{batch}, columns], got {table.dtype} {tuple(table.shape)}")
        if table.shape[1] > 1 and table.stride(1) != 1 or batch > 1 and table.stride(0) < table.shape[1]:
            raise ValueError("rows of the page table must be contiguous and apart")
        if table.device != self.device:
            raise ValueError(f"the page table is on {table.device}, the cache on {self.device}")

    @staticmethod
    def _table_args(table: torch.Tensor) -> tuple[int, int]:
        return max(table.stride(0), table.shape[1]), table.shape[1]

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, *,
               rotary: Rotary | None = None, q: torch.Tensor | None = None,
               seen: torch.dtype | None = None) -> Appended:
        """Write new tokens: k, v [batch, tokens, kv_heads, head_dim], token t of sequence b at position start[b] + t.

        With ``rotary`` the keys are rotated to their positions first, and ``q`` [batch, tokens, heads, head_dim] too,
        into a new tensor.  With ``seen`` the new keys and values come back in that type as the cache holds them.
        Positions outside the table, or whose entry names no page, are not stored.
        """
        sig = (k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype, v.get_device(), table.shape,
               table.stride(), table.dtype, table.get_device(), start.shape, start.stride(), start.dtype,
               start.get_device(), rotary, seen) + (() if q is None else (q.shape, q.stride(), q.dtype, q.get_device()))
        plan = self._plans.get(sig)
        if plan is None:
            plan = self._append_plan(sig, k, v, table, start, rotary, q, seen)
        rot_arg, q_arg, qo_arg, k_arg, v_arg, seen_arg, ld, cols, batch, tokens, index = plan
        q_out = k_out = v_out = None
        q_ptr = qo_ptr = ko_ptr = vo_ptr = None
        if q is not None:
            q_out = q.new_empty(q.shape)
            q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
        if seen is not None:
            k_out, v_out = k.new_empty(k.shape, dtype=seen), k.new_empty(k.shape, dtype=seen)
            ko_ptr, vo_ptr = k_out.data_ptr(), v_out.data_ptr()
        if batch and tokens:
            K.call("tgm_kv_append", self._arg, rot_arg, q_arg, q_ptr, qo_arg, qo_ptr, k_arg, k.data_ptr(), v_arg,
                   v.data_ptr(), seen_arg, ko_ptr, vo_ptr, table.data_ptr(), ld, cols, start.data_ptr(), batch, tokens,
                   K.stream_on(index))
        return Appended(q_out, k_out, v_out)

    def _append_plan(self, sig, k, v, table, start, rotary, q, seen) -> tuple:
        check_heads(k, "k")
        check_heads(v, "v")
        batch, tokens, hk, hd = k.shape
        if hk != self.kv_heads or hd != self.head_dim or v.shape != k.shape:
            raise ValueError(f"k and v must be [batch, tokens, {self.kv_heads}, {self.head_dim}], got {tuple(k.shape)} "
                             f"and {tuple(v.shape)}")
        if v.dtype is not k.dtype or k.device != self.device or v.device != self.device:
            raise ValueError("k and v must be of one type, on the cache's device")
        self._check_table(table, batch)
        check_index(start, "start", batch, k)
        if rotary is not None:
            rotary.check(k, self.head_dim)
        if q is not None:
            check_heads(q, "q")
            if q.shape[:2] != k.shape[:2] or q.shape[2] < 1 or q.shape[3] != hd or q.dtype is not k.dtype or q.device != k.device:
                raise ValueError("q must be [batch, tokens, heads, head_dim] beside k, of its type")
        if seen is not None and seen not in _DT:
            raise ValueError(f"seen must be float32, float16 or bfloat16, got {seen}")
        K.require_device(k)

        def fresh(heads: int, dtype: torch.dtype) -> bytes:
            return _HEADS(tokens * heads * hd, heads * hd, hd, heads, _DT[dtype])

        ld, cols = self._table_args(table)
        return self._plans.keep(sig, (None if rotary is None else rotary.arg, None if q is None else heads_arg(q),
                                      None if q is None else fresh(q.shape[2], q.dtype), heads_arg(k), heads_arg(v),
                                      None if seen is None else fresh(hk, seen), ld, cols, batch, tokens, k.get_device()))

    def read(self, table: torch.Tensor, first: torch.Tensor, count: int,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of positions first[b] .. first[b] + count - 1, each [batch, count, kv_heads, head_dim].

        Positions that no page holds read as zeros."""
        batch = table.shape[0] if table.dim() == 2 else 0
        self._check_table(table, batch)
        check_index(first, "first", batch, table)
        if dtype not in _DT:
            raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        if count < 0:
            raise ValueError("count must not be negative")
        K.require_device(self.k_data)
        shape = (batch, count, self.kv_heads, self.head_dim)
        k, v = torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device)
        if not batch or not count:
            return k, v
        K.call("tgm_kv_read", self._arg, table.data_ptr(), *self._table_args(table), first.data_ptr(), batch, count, k.data_ptr(),
               v.data_ptr(), _DT[dtype], K.stream_of(table))
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *, shared: int = 0,
               scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the newest tokens: q [batch, tokens, heads, head_dim] (rotated), out alike; ``out``, if given, is
        contiguous, and q itself or memory that the two do not share.

        ``lengths`` (int32 [batch]) counts the cached positions of each sequence with the new tokens among them: token
        t of sequence b sees positions 0 .. lengths[b] - tokens + t; a token that sees none gives zeros, one whose scores
        hold a NaN or +infinity gives NaN.  Query head h reads kv head h // (heads // kv_heads).  Scores are multiplied by
        ``scale`` (1 / sqrt(head_dim)).

        ``shared`` positions (a multiple of page_size) from the front are common to the batch: they lie in the pages
        that row 0 of the table names, and are read once for all sequences.
        """
        scale = self._scale if scale is None else float(scale)
        if not 0 < scale < 1e30:
            raise ValueError(f"scale must be positive, got {scale}")
        if out is not None and (out.shape != q.shape or out.dtype is not q.dtype or out.device != q.device
                                or not out.is_contiguous()):
            raise ValueError("out must be like q, and contiguous")
        sig = (q.shape, q.stride(), q.dtype, q.get_device(), table.shape, table.stride(), table.dtype, table.get_device(),
               lengths.shape, lengths.stride(), lengths.dtype, lengths.get_device(), shared)
        plan = self._plans.get(sig)
        if plan is None:
            plan = self._attend_plan(sig, q, table, lengths, shared)
        q_arg, ld, cols, batch, tokens, need, index = plan
        if out is None:
            out = q.new_empty(q.shape)
        else:
            out_sig = (q.shape, q.stride(), q.dtype)
            (self._plans.get(out_sig) or self._plans.keep(out_sig, OutLayout(out, q))).check(out, q, "q")
        # the workspace is of the caching allocator, so that calls on several streams never share one; held until the
        # launch, or another thread's call on this stream could be given its memory before that
        workspace = q.new_empty(need, dtype=torch.uint8) if need else None
        if batch and tokens:
            K.call("tgm_kv_attend", self._arg, q_arg, q.data_ptr(), table.data_ptr(), ld, cols, lengths.data_ptr(), batch,
                   tokens, shared, scale, K.ptr(workspace), need, out.data_ptr(), K.stream_on(index))
        return out

    def _attend_plan(self, sig, q, table, lengths, shared) -> tuple:
        check_heads(q, "q")
        batch, tokens, heads, head_dim = q.shape
        if head_dim != self.head_dim or heads < 1 or heads % self.kv_heads:
            raise ValueError(f"q must have heads of {self.head_dim} values, a multiple of {self.kv_heads} of them, got "
                             f"{tuple(q.shape)}")
        if q.device != self.device:
            raise ValueError(f"q is on {q.device}, the cache on {self.device}")
        self._check_table(table, batch)
        check_index(lengths, "lengths", batch, q)
        if shared < 0 or shared % self.page_size or shared > table.shape[1] * self.page_size:
            raise ValueError(f"shared must be a multiple of {self.page_size} within the page table, got {shared}")
        K.require_device(q)
        ld, cols = self._table_args(table)
        need = K.load_library().tgm_kv_attend_workspace(self._arg, _DT[q.dtype], heads, batch, tokens, cols, shared)
        return self._plans.keep(sig, (heads_arg(q), ld, cols, batch, tokens, need, q.get_device()))
