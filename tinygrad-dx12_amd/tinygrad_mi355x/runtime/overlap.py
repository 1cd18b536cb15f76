"""Which strided tensors share memory: what an operator that is given its output tensor has to know before it launches.

Exact, not by the tensors' ranges: the outputs of a serving loop are often heads of stacked rows, whose ranges lie inside
each other.  Two elements meet where a sum of strides times index differences is the distance of the tensors' addresses;
that is searched from the largest stride down, where nearly every step leaves one or two differences to try.
"""

from __future__ import annotations

import torch


def _reaches(delta: int, spans: list[tuple[int, int, int]]) -> bool:
    """Whether delta is a sum of c * stride over ``spans`` (stride, lowest c, highest c), strides positive and descending."""
    if not spans:
        return delta == 0
    (stride, lowest, highest), rest = spans[0], spans[1:]
    low, high = sum(s * a for s, a, _ in rest), sum(s * b for s, _, b in rest)
    first, last = max(lowest, -((high - delta) // stride)), min(highest, (delta - low) // stride)
    return any(_reaches(delta - c * stride, rest) for c in range(first, last + 1))


def _spans(t: torch.Tensor) -> list[tuple[int, int]]:
    """(bytes apart, highest index) of the dimensions of ``t`` with more than one index, the widest first."""
    return sorted(((s * t.element_size(), n - 1) for s, n in zip(t.stride(), t.shape) if n > 1), reverse=True)


def overlaps_itself(t: torch.Tensor) -> bool:
    """Whether two elements of ``t`` share memory."""
    spans = _spans(t)
    if not t.numel() or not spans:
        return False
    if spans[-1][0] == 0:
        return True
    signed = [(s, -n, n) for s, n in spans]
    return any(_reaches(-c * s, signed[i + 1:]) for i, (s, n) in enumerate(spans)
               for c in range(1, min(n, sum(a * b for a, b in spans[i + 1:]) // s) + 1))


def _extent(t: torch.Tensor, spans: list[tuple[int, int]]) -> int:
    """Bytes from the first element to the end of the last."""
    return sum(s * n for s, n in spans) + t.element_size() if t.numel() else 0


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether an element of ``a`` and one of ``b`` share memory."""
    delta, at, bt = b.data_ptr() - a.data_ptr(), _spans(a), _spans(b)
    if not a.numel() or not b.numel() or not -_extent(b, bt) < delta < _extent(a, at):
        return False
    spans = {1: [1 - b.element_size(), a.element_size() - 1]}  # the bytes of an element
    for s, n in at:
        spans.setdefault(s, [0, 0])[1] += n
    for s, n in bt:
        spans.setdefault(s, [0, 0])[0] -= n
    spans.pop(0, None)  # expanded dimensions
    return _reaches(delta, [(s, *spans[s]) for s in sorted(spans, reverse=True)])


class OutLayout:
    """What the layouts of an operator's ``out`` and of the input ``x`` (of its shape and type) say about the memory that
    the two share, for calls with any addresses: elements are read and written in no order."""

    def __init__(self, out: torch.Tensor, x: torch.Tensor) -> None:
        if overlaps_itself(out):
            raise ValueError("elements of out must not share memory")
        self.same = all(s == t for s, t, n in zip(out.stride(), x.stride(), x.shape) if n > 1)
        self.before, self.behind = -_extent(out, _spans(out)), _extent(x, _spans(x))

    def check(self, out: torch.Tensor, x: torch.Tensor, name: str) -> None:
        """Refuses an ``out`` that shares memory with ``x`` without being ``x``."""
        delta = out.data_ptr() - x.data_ptr()
        if self.before < delta < self.behind and not (self.same and delta == 0) and overlap(x, out):
            raise ValueError(f"out must be {name} itself or share no memory with it")
