"""Cross-entropy loss of an output head  z = x W  with its gradients, without the logits in memory.  Native kernels for CUDA tensors,
fp32 formulation for CPU tensors.

    loss_t = log sum_v exp(z_tv) - z_t,y      dz = scale (softmax(z) - onehot y)      dx = dz W^T      dW = x^T dz

The weight lies as [inputs, columns] (layout 'nn') or [columns, inputs] ('nt', as an embedding table); columns from ``vocab`` on are
padding: they have no probability and their gradient is 0.  A target outside [0, vocab) is no label: loss and gradient of the token are 0.

On a GPU the product's epilogue takes the maximum of every row over the 128 or 256 columns of a tile from the fp32 sums, and the sum of
the exponentials relative to it; the joined maxima and sums give the loss.  For the gradient the exponentials are kept for some rows
at a time, become dz where they lie, and go into the two products of the gradients.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native
from . import rows as _rows
from .gemm import gemm_pair, sm_count

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
    if w.dtype != x.dtype or w.device != x.device or targets.device != x.device:
        raise ValueError(f"x is {x.dtype} on {x.device}, the weight {w.dtype} on {w.device}, targets on {targets.device}")
    if x.is_cuda:
        if x.dtype != torch.bfloat16:
            raise ValueError(f"the kernels need bf16 (got {x.dtype})")
        if d % 8 or (layout == "nn" and cols % 8):
            raise ValueError(f"the kernels need rows of a multiple of 8 elements (got {d} inputs, {cols} columns, {layout})")
        if n >= 1 << 31 or cols > 1 << 20:
            raise ValueError(f"the kernels take fewer than 2^31 tokens and at most 2^20 columns (got {n}, {cols})")
        _native.check_device(x)
    return n, d, cols


def _partial(x, w, targets, vocab: int, layout: str, e, columns: int, stats, label, tile_n: int):
    _native.load().head_partial(x.shape[0], x.shape[1], vocab, columns, x.data_ptr(), _rows.pitch(x), w.data_ptr(), _rows.pitch(w),
                                1 if layout == "nn" else 0, 0 if e is None else e.data_ptr(), columns, stats.data_ptr(), label.data_ptr(),
                                targets.data_ptr(), tile_n, sm_count(x.device), _native.status().dev, _native.stream_ptr())


def _join(e, columns: int, stats, label, targets, vocab: int, tile_n: int, scale: float, loss):
    _native.load().head_rows(0 if e is None else e.data_ptr(), columns, stats.data_ptr(), label.data_ptr(), targets.data_ptr(),
                             targets.shape[0], columns, stats.shape[0], tile_n, vocab, scale, loss.data_ptr(), _native.stream_ptr())


def _plan(n: int, columns: int, device) -> int:
    C = _native.load()
    return C.products_tile_n(C.PRODUCT_HEAD, n, columns, 1, sm_count(device))


def head_loss(x, w, targets, vocab: int, layout: str = "nn") -> torch.Tensor:
    """Loss [tokens] (fp32) of ``x`` [tokens, inputs] under the head ``w``."""
    n, _, _ = _check(x, w, targets, vocab, layout)
    if not x.is_cuda:
        return _reference(x, w, targets, vocab, layout)[0]
    loss = torch.empty(n, dtype=torch.float32, device=x.device)
    if n:
        x, w, targets = _rows.as_aligned(x), _rows.as_aligned(w), targets.contiguous()
        tile_n = _plan(n, vocab, x.device)
        stats = torch.empty(-(-vocab // tile_n), n, 2, dtype=torch.float32, device=x.device)
        label = torch.empty(n, dtype=torch.float32, device=x.device)
        _partial(x, w, targets, vocab, layout, None, vocab, stats, label, tile_n)
        _join(None, 0, stats, label, targets, vocab, tile_n, 0.0, loss)
    return loss


def head_loss_grad(x, w, targets, vocab: int, scale: float, layout: str = "nn", dw: Optional[torch.Tensor] = None, rows: int = 0):
    """(loss [tokens] in fp32 and not scaled, dx, dw): the gradients times ``scale``.  ``dw`` (fp32 or the weight's type, the weight's
    layout) is added to; without it the weight's gradient is a new tensor.  ``rows``: tokens whose exponentials are in memory at a
    time (0: as many as half a gigabyte holds)."""
    n, d, cols = _check(x, w, targets, vocab, layout)
    if rows < 0:
        raise ValueError(f"rows at a time are not negative (got {rows})")
    add = dw is not None
    if add:
        if dw.shape != w.shape or dw.device != w.device or dw.dtype not in (torch.float32, w.dtype):
            raise ValueError(f"dw must be fp32 or {w.dtype} {tuple(w.shape)} on {w.device} (got {dw.dtype} {tuple(dw.shape)} on {dw.device})")
        if x.is_cuda and not (_rows.aligned(dw) and _rows.pitch(dw) % 8 == 0):
            raise ValueError("a gradient that is added to needs neighbouring columns and rows on 16-byte boundaries")
    if not x.is_cuda:
        loss, dz = _reference(x, w, targets, vocab, layout, scale)
        dx = dz @ (w.float().T if layout == "nn" else w.float())
        new = x.float().T @ dz if layout == "nn" else dz.T @ x.float()
        if not add:
            return loss, dx.to(x.dtype), new.to(w.dtype)
        dw += new.to(dw.dtype)
        return loss, dx.to(x.dtype), dw
    loss = torch.empty(n, dtype=torch.float32, device=x.device)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if n == 0:
        return loss, dx, dw if add else torch.zeros(w.shape, dtype=w.dtype, device=w.device)
    x, w, targets = _rows.as_aligned(x), _rows.as_aligned(w), targets.contiguous()
    columns = -(-vocab // 64) * 64                        # of the exponentials: zeros from vocab on
    wide = min(columns, cols)                             # those of the weight's gradient that a product writes
    most = rows or max(256, PIECE_BYTES // (2 * columns) // 256 * 256)
    pieces = -(-n // most)
    piece = min(n, rows or -(-n // pieces // 256) * 256)     # equal ones, of whole tiles
    tile_n = _plan(piece, columns, x.device)
    e = torch.empty(piece, columns, dtype=x.dtype, device=x.device)
    stats = torch.empty(-(-columns // tile_n) * piece * 2, dtype=torch.float32, device=x.device)
    label = torch.empty(piece, dtype=torch.float32, device=x.device)
    if not add:
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device)
    # sums over several pieces are held in fp32
    total = dw if dw.dtype == torch.float32 or pieces == 1 else torch.empty(w.shape, dtype=torch.float32, device=w.device)
    part = (lambda t: t[:, :wide]) if layout == "nn" else (lambda t: t[:wide])
    given, known = (w[:, :vocab], "nt") if layout == "nn" else (w[:vocab], "nn")
    for k, i in enumerate(range(0, n, piece)):
        xi, ti = x[i:i + piece], targets[i:i + piece]
        m = xi.shape[0]
        ei, si = e[:m], stats[:-(-columns // tile_n) * m * 2].view(-1, m, 2)
        _partial(xi, w, ti, vocab, layout, ei, columns, si, label, tile_n)
        _join(ei, columns, si, label, ti, vocab, tile_n, scale, loss[i:i + piece])
        first = (xi, ei[:, :wide], "tn") if layout == "nn" else (ei[:, :wide], xi, "tn")
        gemm_pair(*first, part(total), k > 0 or (add and total is dw), ei[:, :vocab], given, known, dx[i:i + piece])
    if wide < cols and not (add and total is dw):
        (total[:, wide:] if layout == "nn" else total[wide:]).zero_()
    if total is not dw:
        if dw.is_contiguous() and dw.numel() % 4 == 0:
            _native.load().cast_f32_to_bf16(total.data_ptr(), dw.data_ptr(), dw.numel(), 1 if add else 0, _native.stream_ptr())
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
