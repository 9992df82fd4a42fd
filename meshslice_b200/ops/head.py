"""Cross-entropy loss of an output head  z = x W  with its gradients, without the logits in memory.  Native kernels for CUDA tensors,
fp32 formulation for CPU tensors.

    loss_t = log sum_v exp(z_tv) - z_t,y      dz = scale (softmax(z) - onehot y)      dx = dz W^T      dW = x^T dz

The weight lies as [inputs, columns] (layout 'nn') or [columns, inputs] ('nt', as an embedding table); columns from ``vocab`` on are
padding: they have no probability and their gradient is 0.  A target outside [0, vocab) is no label: loss and gradient of the token are 0.

On a GPU the product's epilogue takes the maximum of every row over half the columns of a tile, 64 or 128, from the fp32 sums, and the sum of
the exponentials relative to it; the joined maxima and sums give the loss.  For the gradient the exponentials are kept for some rows
at a time, become dz where they lie, and go into the two products of the gradients.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native
from . import rows as _rows
from .gemm import _SM_COUNT, sm_count

PIECE_BYTES = 1 << 29      # of exponentials that are in memory at a time, unless the caller says how many rows


def _check(x, w, targets, vocab: int, layout: str) -> Tuple[int, int, int]:
    """(tokens, inputs, columns)"""
    if layout not in ("nn", "nt"):
        raise ValueError(f"the weight lies as 'nn' or 'nt' (got {layout!r})")
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError(f"x and the weight are matrices (got {tuple(x.shape)}, {tuple(w.shape)})")
    n, d = x.shape
    i, cols = w.shape if layout == "nn" else w.shape[::-1]
    if i != d or d < 1:
        raise ValueError(f"shapes do not fit: x {tuple(x.shape)}, weight {tuple(w.shape)} ({layout})")
    if not 0 < vocab <= cols:
        raise ValueError(f"the vocabulary must have a token, and at most the weight's {cols} columns (got {vocab})")
    if targets.shape != (n,) or targets.dtype != torch.int64:
        raise ValueError(f"targets must be int64 [{n}] (got {targets.dtype} {tuple(targets.shape)})")
    if w.dtype is not x.dtype or w.get_device() != x.get_device() or targets.get_device() != x.get_device():
        raise ValueError(f"x is {x.dtype} on {x.device}, the weight {w.dtype} on {w.device}, targets on {targets.device}")
    if x.is_cuda:
        if x.dtype != torch.bfloat16:
            raise ValueError(f"the kernels need bf16 (got {x.dtype})")
        if d % 8 or (layout == "nn" and cols % 8):
            raise ValueError(f"the kernels need rows of a multiple of 8 elements (got {d} inputs, {cols} columns, {layout})")
        if n >= 1 << 31 or vocab > 1 << 18:
            raise ValueError(f"the kernels take fewer than 2^31 tokens and a vocabulary of at most 2^18 (got {n}, {vocab})")
        _native.check_device(x)
    return n, d, cols


def _tile_n(n: int, columns: int, sms: int) -> int:
    C = _native.load()
    return C.products_tile_n(C.PRODUCT_HEAD, n, columns, 1, sms)


def _at(t, pitch: int):
    """(tensor, address, row pitch) as the kernels take a matrix whose rows are ``pitch`` long; a copy where they cannot address it."""
    if t.is_contiguous():
        p = t.data_ptr()
        if p & 15 == 0:
            return t, p, pitch
    t = _rows.as_aligned(t)
    return t, t.data_ptr(), _rows.pitch(t)


def head_loss(x, w, targets, vocab: int, layout: str = "nn") -> torch.Tensor:
    """Loss [tokens] (fp32) of ``x`` [tokens, inputs] under the head ``w``."""
    n, d, cols = _check(x, w, targets, vocab, layout)
    if not x.is_cuda:
        return _reference(x, w, targets, vocab, layout)[0]
    loss = torch.empty(n, dtype=torch.float32, device=x.device)
    if n:
        x, px, lx = _at(x, d)
        w, pw, lw = _at(w, cols if layout == "nn" else d)
        targets = targets.contiguous()
        sms = _SM_COUNT.get(x.get_device()) or sm_count(x.device)
        tile_n = _tile_n(n, vocab, sms)
        blocks = -(-vocab * 2 // tile_n)                  # statistics are of half a tile's columns
        space = torch.empty((2 * blocks + 1) * n, dtype=torch.float32, device=x.device)
        at = space.data_ptr()
        _native.load().head_losses(n, d, vocab, px, lx, pw, lw, 1 if layout == "nt" else 0,
                                   targets.data_ptr(), at, at + 8 * blocks * n, tile_n, loss.data_ptr(), sms, _native.status().dev,
                                   _native.stream_ptr())
    return loss


def head_loss_grad(x, w, targets, vocab: int, scale: float, layout: str = "nn", dw: Optional[torch.Tensor] = None, rows: int = 0):
    """(loss [tokens] in fp32 and not scaled, dx, dw): the gradients times ``scale``.  ``dw`` (fp32 or the weight's type, the weight's
    layout) is added to and shares no memory with an operand; without it the weight's gradient is a new tensor.  ``rows``: tokens whose
    exponentials are in memory at a time (0: as many as half a gigabyte holds)."""
    n, d, cols = _check(x, w, targets, vocab, layout)
    if rows < 0:
        raise ValueError(f"rows at a time are not negative (got {rows})")
    add = dw is not None
    if add:
        if dw.shape != w.shape or dw.device != w.device or dw.dtype not in (torch.float32, w.dtype):
            raise ValueError(f"dw must be fp32 or {w.dtype} {tuple(w.shape)} on {w.device} (got {dw.dtype} {tuple(dw.shape)} on {dw.device})")
        if x.is_cuda and not _rows.adds(dw):
            raise ValueError("a gradient that is added to needs neighbouring columns and rows on 16-byte boundaries")
        _rows.check_apart((dw,), (x, w, targets), "dw")       # pieces of the tokens read the operands after others were added
    if not x.is_cuda:
        loss, dz = _reference(x, w, targets, vocab, layout, scale)
        dx = dz @ (w.float().T if layout == "nn" else w.float())
        new = x.float().T @ dz if layout == "nn" else dz.T @ x.float()
        if not add:
            return loss, dx.to(x.dtype), new.to(w.dtype)
        dw += new.to(dw.dtype)
        return loss, dx.to(x.dtype), dw
    loss = torch.empty(n, dtype=torch.float32, device=x.device)
    dx = x.new_empty(n, d)
    if n == 0:
        return loss, dx, dw if add else torch.zeros(w.shape, dtype=w.dtype, device=w.device)
    nt = layout == "nt"
    x, px, lx = _at(x, d)
    w, pw, lw = _at(w, d if nt else cols)
    targets = targets.contiguous()
    columns = -(-vocab // 64) * 64                        # of the exponentials: zeros from vocab on
    wide = min(columns, cols)                             # those of the weight's gradient that a product writes
    if not add:
        dw = w.new_empty(w.shape)
    # Sums over several pieces are held in fp32; where that would take a matrix of its own, as much memory is better spent on a larger piece.
    limit = PIECE_BYTES + (0 if dw.dtype is torch.float32 else 4 * w.numel())
    most = rows or max(256, limit // (2 * columns) // 256 * 256)
    if not rows and most < n:
        most = max(256, PIECE_BYTES // (2 * columns) // 256 * 256)
    pieces = -(-n // most)
    piece = min(n, rows or -(-n // pieces // 256) * 256)     # equal ones, of whole tiles
    total = dw if dw.dtype is torch.float32 or piece == n else torch.empty(w.shape, dtype=torch.float32, device=w.device)
    C, sms, status, stream = _native.load(), _SM_COUNT.get(x.get_device()) or sm_count(x.device), _native.status().dev, _native.stream_ptr()
    tile_n = _tile_n(piece, columns, sms)
    blocks = -(-columns * 2 // tile_n)
    parts = C.head_parts(piece, d, vocab, sms)            # of the tokens' gradient, held in fp32 beside the others
    sums = -(-piece // 32) * 32 * d * parts if parts > 1 else 0
    space = x.new_empty((columns + 4 * blocks + 2) * piece + 2 * sums + 8)
    e = space.data_ptr()
    stats, label = e + 2 * columns * piece, e + (2 * columns + 8 * blocks) * piece
    partial = (label + 4 * piece + 15) // 16 * 16
    pitch, size = _rows.pitch(total) if add else (d if nt else cols), total.element_size()
    at, fp32, onto = total.data_ptr(), 1 if size == 4 else 0, add and total is dw
    pad = (0, 0, 0, 0)
    if wide < cols and not onto:
        pad = (at + size * wide * pitch, size * pitch, size * d, cols - wide) if nt else (at + size * wide, size * pitch, size * (cols - wide), d)
    for i in range(0, n, piece):
        C.head_grads(min(piece, n - i), d, vocab, columns, wide, px + 2 * i * lx, lx, pw, lw, 1 if nt else 0, targets.data_ptr() + 8 * i, scale, e,
                     stats, label, tile_n, loss.data_ptr() + 4 * i, dx.data_ptr() + 2 * i * d, at, pitch, fp32, 1 if i or onto else 0, parts, partial,
                     *(pad if i == 0 else (0, 0, 0, 0)), sms, status, stream)
    if total is not dw:
        if dw.is_contiguous() and dw.numel() % 4 == 0:
            C.cast_f32_to_bf16(total.data_ptr(), dw.data_ptr(), dw.numel(), 1 if add else 0, stream)
        elif add:
            dw += total
        else:
            dw.copy_(total)
    return loss, dx, dw


def _reference(x, w, targets, vocab: int, layout: str, scale: Optional[float] = None):
    """(loss, dz [tokens, columns] with ``scale``)"""
    z = x.float() @ (w.float() if layout == "nn" else w.float().T)
    label = (targets >= 0) & (targets < vocab)
    y = torch.where(label, targets, 0)[:, None]
    logp = torch.log_softmax(z[:, :vocab], 1)
    loss = torch.where(label, -logp.gather(1, y)[:, 0], 0.0)
    if scale is None:
        return loss, None
    dz = torch.zeros_like(z)
    dz[:, :vocab] = torch.where(label[:, None], logp.exp() * scale, 0.0)
    dz.scatter_add_(1, y, torch.where(label, -scale, 0.0)[:, None])
    return loss, dz
