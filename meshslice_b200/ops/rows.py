"""How the kernels that take a row pitch address a matrix: neighbouring columns, rows on 16-byte boundaries."""
from __future__ import annotations

import torch


def pitch(t) -> int:
    """Elements from one row to the next (that of a single row is never used: its length)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def aligned(t) -> bool:
    return ((t.shape[1] <= 1 or t.stride(1) == 1) and pitch(t) >= t.shape[1] and pitch(t) * t.element_size() % 16 == 0
            and t.data_ptr() % 16 == 0)


def adds(t) -> bool:
    """The kernels can add to ``t``: rows of multiples of 8 elements apart, on 16-byte boundaries."""
    if t.is_contiguous():
        return t.data_ptr() & 15 == 0 and t.shape[1] % 8 == 0
    return aligned(t) and pitch(t) % 8 == 0


def as_aligned(t):
    """``t``, or a copy of it where the kernels cannot address it."""
    return t if aligned(t) else t.clone(memory_format=torch.contiguous_format)


def overlap(a, b) -> bool:
    """The memory of two matrices with ``aligned`` rows has a byte in common (or may have)."""
    span = lambda t: (t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * pitch(t) + t.shape[1]) * t.element_size())
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _span(t):
    """Addresses of the first byte and of the one behind the last."""
    p = t.data_ptr()
    if t.is_contiguous():
        return p, p + t.nbytes
    return p, p + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0)


def _lines(t):
    """(bytes from the first to the last element of a line, bytes from one line to the next, lines) of a matrix or vector, along the
    dimension of the smaller stride."""
    dims = sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1 and s > 0)
    size = t.element_size()
    inner, outer = dims[0] if dims else (0, 1), dims[1] if len(dims) > 1 else (0, 1)
    return size * (1 + inner[0] * (inner[1] - 1)), size * outer[0], outer[1]


def meet(a, b) -> bool:
    """The memory of two matrices or vectors has a byte in common (or may have).  Columns of one wider matrix that lie side by side do not
    meet."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if not (a0 < b1 and b0 < a1):
        return False
    (wa, pa, na), (wb, pb, nb) = _lines(a), _lines(b)
    pitch = pa if na > 1 else pb
    if (na > 1 and nb > 1 and pa != pb) or na == nb == 1 or wa > pitch or wb > pitch:
        return True
    at = (b0 - a0) % pitch                       # of b's lines, counted from where a's begin
    return at < wa or at + wb > pitch


def check_apart(written, read, what: str):
    """Refuses tensors that a kernel writes while it writes or reads another one there."""
    n = len(written)
    spans = [(*_span(t), i < n) for i, t in enumerate((*written, *read))]
    spans.sort()
    end_written = end = 0
    for first, last, writes in spans:
        if first < (end if writes else end_written):
            break
        if last > end:
            end = last
        if writes:
            end_written = last
    else:
        return
    for i, t in enumerate(written):
        if any(meet(t, o) for o in (*written[i + 1:], *read)):
            raise ValueError(f"{what} shares memory with another one or with an operand")
