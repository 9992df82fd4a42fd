"""How the kernels that take a row pitch address a matrix: neighbouring columns, rows on 16-byte boundaries."""
from __future__ import annotations

import torch


def pitch(t) -> int:
    """Elements from one row to the next (that of a single row is never used: its length)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def aligned(t) -> bool:
    return ((t.shape[1] <= 1 or t.stride(1) == 1) and pitch(t) >= t.shape[1] and pitch(t) * t.element_size() % 16 == 0
            and t.data_ptr() % 16 == 0)


def as_aligned(t):
    """``t``, or a copy of it where the kernels cannot address it."""
    return t if aligned(t) else t.clone(memory_format=torch.contiguous_format)


def overlap(a, b) -> bool:
    """The memory of two matrices with ``aligned`` rows has a byte in common (or may have)."""
    span = lambda t: (t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * pitch(t) + t.shape[1]) * t.element_size())
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1
