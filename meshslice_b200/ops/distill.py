"""Distillation loss of rows of logits from a teacher's top logits, with its gradient.  Native kernels for CUDA tensors, fp32
formulation for CPU tensors.

Per row, with z the student's logits over the vocabulary, p = softmax(t / T) over the teacher's entries, y the label:

    loss = w (log sum exp z - z_y) + (1 - w) T^2 sum_k p_k (log p_k - log softmax(z / T) at id_k)
    d loss / d z = w (softmax z - onehot y) + (1 - w) T (softmax(z / T) - p)

The second term is KL(p || softmax(z / T)) where every id occurs once.  Entries that share an id count as an event each: beside one entry of
their joint probability the loss is lower by (1 - w) T^2 times what they are uncertain among themselves, which depends on the teacher alone
(so the loss may be negative); the gradient is the same.

An id outside [0, vocab) is no entry (teachers that kept fewer than others), a target outside is no label; a term without entries or
label is zero, in the loss and in the gradient.  T^2 keeps the gradient's size as T grows.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .. import _native
from . import rows


_VALUES = {torch.float32: 0, torch.bfloat16: 1}     # types of the teacher's logits


def _check(logits, ids, values, vocab: int, temperature: float, targets, hard_weight: float):
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, columns] (got {tuple(logits.shape)})")
    n = logits.shape[0]
    if ids.dim() != 2 or ids.shape[0] != n or ids.dtype != torch.int64:
        raise ValueError(f"teacher ids must be int64 [rows, top] (got {ids.dtype} {tuple(ids.shape)})")
    if values.shape != ids.shape or values.dtype not in _VALUES:
        raise ValueError(f"teacher logits must be fp32 or bf16 of the ids' shape (got {values.dtype} {tuple(values.shape)})")
    if targets is not None and (targets.shape != (n,) or targets.dtype != torch.int64):
        raise ValueError(f"targets must be int64 [rows] (got {targets.dtype} {tuple(targets.shape)})")
    if targets is None and hard_weight != 0.0:
        raise ValueError("a hard weight needs targets")
    if vocab < 1:
        raise ValueError(f"the vocabulary must have a token (got {vocab})")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"the temperature must be positive and finite (got {temperature})")
    if not 0.0 <= hard_weight <= 1.0:
        raise ValueError(f"the hard weight must be in [0, 1] (got {hard_weight})")
    for t in (ids, values, targets):
        if t is not None and t.device != logits.device:
            raise ValueError(f"logits are on {logits.device}, other inputs on {t.device}")
    if logits.is_cuda:
        if logits.dtype != torch.bfloat16 or logits.shape[1] % 8:
            raise ValueError(f"the kernels need bf16 logits of a multiple of 8 columns (got {logits.dtype} {tuple(logits.shape)})")
        if ids.shape[1] > _native.load().DISTILL_TOP:
            raise ValueError(f"at most {_native.load().DISTILL_TOP} teacher entries per row (got {ids.shape[1]})")
        _native.check_device(logits)


def _gradient_to(logits, out):
    """Where the kernels write the gradient: ``out``, a new tensor, or one that is copied to ``out`` afterwards."""
    if out is None:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must have the logits' shape, type and device")
    same = out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()
    if not logits.is_cuda or (rows.aligned(out) and (same or not rows.aligned(logits) or not rows.overlap(out, logits))):
        return out
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


def _launch(step: int, logits, grad, ids, values, targets, col_offset: int, vocab: int, temperature: float, hard_weight: float,
            scale: float, loss, stats):
    z = grad if grad is not None and grad.data_ptr() == logits.data_ptr() else rows.as_aligned(logits)
    ids, values = ids.contiguous(), values.contiguous()
    targets = None if targets is None else targets.contiguous()
    p = lambda t: 0 if t is None else t.data_ptr()
    _native.load().distill(step, z.data_ptr(), rows.pitch(z), p(grad), 0 if grad is None else rows.pitch(grad), ids.data_ptr(),
                           values.data_ptr(), _VALUES[values.dtype], p(targets), z.shape[0], z.shape[1], col_offset,
                           vocab, ids.shape[1], temperature, hard_weight, scale, p(loss), p(stats), _native.stream_ptr())


def distill_loss_grad(logits, teacher_ids, teacher_logits, vocab: int, scale: float, temperature: float = 1.0, targets=None,
                      hard_weight: float = 0.0, out=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Loss [rows] (fp32, not scaled) and gradient times ``scale`` of whole rows of logits [rows, columns >= vocab]; columns from
    ``vocab`` on are padding and get 0.  ``teacher_ids`` int64 and ``teacher_logits`` fp32 or bf16 [rows, top].  The gradient goes to
    ``out`` (``out=logits`` works in place) or a new tensor."""
    # the common call, checked in a few steps: a kernel of a few us is over before a longer list of them
    if (logits.is_cuda and out is None and logits.dtype is torch.bfloat16 and logits.dim() == 2 and logits.is_contiguous()
            and teacher_ids.dtype is torch.int64 and teacher_ids.dim() == 2 and teacher_ids.is_contiguous()
            and teacher_logits.dtype in _VALUES and teacher_logits.is_contiguous() and 0.0 <= hard_weight <= 1.0
            and 0.0 < temperature < math.inf):
        n, cols = logits.shape
        shape, dev, z, C = teacher_ids.shape, logits.get_device(), logits.data_ptr(), _native.load()
        top = shape[1]
        if targets is None:
            y, fine = 0, hard_weight == 0.0
        else:
            y, fine = targets.data_ptr(), (targets.dtype is torch.int64 and targets.dim() == 1 and targets.shape[0] == n
                                           and targets.is_contiguous() and targets.get_device() == dev)
        if (fine and shape[0] == n > 0 and teacher_logits.shape == shape and teacher_ids.get_device() == dev == teacher_logits.get_device()
                and cols % 8 == 0 and z & 15 == 0 and 0 < vocab <= cols and vocab <= C.DISTILL_ROW_COLS and top <= C.DISTILL_TOP):
            stream = _native.stream_on(dev)
            grad, loss = torch.empty_like(logits), torch.empty(n, dtype=torch.float32, device=logits.device)
            C.distill(0, z, cols, grad.data_ptr(), cols, teacher_ids.data_ptr(), teacher_logits.data_ptr(), _VALUES[teacher_logits.dtype],
                      y, n, cols, 0, vocab, top, temperature, hard_weight, scale, loss.data_ptr(), 0, stream)
            return loss, grad
    _check(logits, teacher_ids, teacher_logits, vocab, temperature, targets, hard_weight)
    if logits.shape[1] < vocab:
        raise ValueError(f"whole rows have at least vocab = {vocab} columns (got {logits.shape[1]})")
    if not logits.is_cuda or vocab > _native.load().DISTILL_ROW_COLS:
        stats = distill_partial(logits, teacher_ids, teacher_logits, 0, vocab, temperature, targets)
        return distill_grad(logits, teacher_ids, teacher_logits, 0, vocab, scale, stats, temperature, targets, hard_weight, out)
    grad = _gradient_to(logits, out)
    loss = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
    if logits.shape[0]:
        _launch(0, logits, grad, teacher_ids, teacher_logits, targets, 0, vocab, temperature, hard_weight, scale, loss, None)
    if out is not None and grad is not out:
        grad = out.copy_(grad)
    return loss, grad


def _entries(ids, values, vocab: int, temperature: float):
    """Teacher probabilities [rows, top] (0 where there is no entry), ids with 0 in those places, rows that have any."""
    there = (ids >= 0) & (ids < vocab) & (values.float() != -math.inf)
    t = torch.where(there, values.float(), -math.inf)
    lead = t.amax(1, keepdim=True) if ids.shape[1] else t.new_zeros(t.shape[0], 1)
    e = torch.where(there, torch.exp((t - lead) / temperature), 0.0)
    total = e.sum(1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total), torch.where(there, ids, 0), there.any(1)


def distill_partial(logits, teacher_ids, teacher_logits, col_offset: int, vocab: int, temperature: float = 1.0, targets=None):
    """Statistics [rows, 5] of the slice [col_offset, col_offset + columns) of the vocabulary: max, sum exp(z - max),
    sum exp((z - max) / T), sum p z and the label's logit (0 where it is elsewhere)."""
    _check(logits, teacher_ids, teacher_logits, vocab, temperature, targets, 0.0)
    n, cols = logits.shape
    if col_offset < 0:
        raise ValueError(f"the slice starts at a column of the vocabulary (got {col_offset})")
    if logits.is_cuda:
        stats = torch.empty(n, 5, dtype=torch.float32, device=logits.device)
        if n:
            _launch(1, logits, None, teacher_ids, teacher_logits, targets, col_offset, vocab, temperature, 0.0, 0.0, None, stats)
        return stats
    valid = max(0, min(cols, vocab - col_offset))
    if valid == 0:
        stats = torch.zeros(n, 5)
        stats[:, 0] = -math.inf
        return stats
    z = logits.float()[:, :valid]
    p, ids, _ = _entries(teacher_ids, teacher_logits, vocab, temperature)
    here = (p != 0) & (ids >= col_offset) & (ids < col_offset + valid)
    m = z.max(1, keepdim=True).values
    dot = torch.where(here, p * z.gather(1, (ids - col_offset).clamp(0, valid - 1)), 0.0).sum(1)
    zy = torch.zeros(n)
    if targets is not None:
        y = targets - col_offset
        zy = torch.where((y >= 0) & (y < valid), z.gather(1, y.clamp(0, valid - 1)[:, None])[:, 0], 0.0)
    return torch.stack([m[:, 0], torch.exp(z - m).sum(1), torch.exp((z - m) / temperature).sum(1), dot, zy], 1)


def distill_rescale(stats, gmax, temperature: float = 1.0):
    """Statistics of a slice relative to the maximum ``gmax`` [rows] of whole rows: those of all slices then add up (all but the
    first column, which becomes 0)."""
    d = torch.where(stats[:, 0] == -math.inf, -math.inf, stats[:, 0] - gmax)
    return torch.stack([torch.zeros_like(d), stats[:, 1] * torch.exp(d), stats[:, 2] * torch.exp(d / temperature), stats[:, 3], stats[:, 4]], 1)


def distill_grad(logits, teacher_ids, teacher_logits, col_offset: int, vocab: int, scale: float, stats, temperature: float = 1.0,
                 targets=None, hard_weight: float = 0.0, out: Optional[torch.Tensor] = None):
    """Loss [rows] and gradient of a slice, from the statistics [rows, 5] of whole rows."""
    _check(logits, teacher_ids, teacher_logits, vocab, temperature, targets, hard_weight)
    n, cols = logits.shape
    if stats.shape != (n, 5) or stats.dtype != torch.float32 or stats.device != logits.device:
        raise ValueError(f"statistics must be fp32 [rows, 5] beside the logits (got {stats.dtype} {tuple(stats.shape)} on {stats.device})")
    if col_offset < 0:
        raise ValueError(f"the slice starts at a column of the vocabulary (got {col_offset})")
    grad = _gradient_to(logits, out)
    if logits.is_cuda:
        loss = torch.empty(n, dtype=torch.float32, device=logits.device)
        if n:
            _launch(2, logits, grad, teacher_ids, teacher_logits, targets, col_offset, vocab, temperature, hard_weight, scale, loss,
                    stats.contiguous())
        if out is not None and grad is not out:
            grad = out.copy_(grad)
        return loss, grad
    T, w = temperature, hard_weight
    m, hard, soft, dot, zy = stats.unbind(1)
    p, ids, some = _entries(teacher_ids, teacher_logits, vocab, T)
    label = torch.zeros(n, dtype=torch.bool) if targets is None else (targets >= 0) & (targets < vocab)
    plogp = torch.where(p != 0, p * torch.log(torch.where(p != 0, p, 1.0)), 0.0).sum(1)
    loss = torch.zeros(n)
    if w != 1.0:
        # sum p (z - m): of logits far beyond their differences (masks of the type's lowest value) what the sums' rounding cannot tell
        # from 0 is 0
        above = dot - p.sum(1) * m
        far = (m * (math.log2(math.e) / T)).abs() >= 2.0 ** 24
        above = torch.where(far & (above.abs() <= m.abs().clamp_max(torch.finfo(torch.float32).max) * 2.0 ** -18), 0.0, above)
        loss = loss + torch.where(some, (1 - w) * T * (T * (plogp + torch.log(soft)) - above), 0.0)
    if w != 0.0:
        loss = loss + torch.where(label, w * (torch.log(hard) - (zy - m)), 0.0)
    valid = max(0, min(cols, vocab - col_offset))
    z = logits.float()[:, :valid] - m[:, None]
    drop = torch.where(some, (1 - w) * T * scale, 0.0)
    mark = torch.where(label, w * scale, 0.0)
    g = torch.zeros(n, cols)
    learnt = ((drop != 0) | (mark != 0))[:, None]
    g[:, :valid] = torch.where(learnt, torch.exp(z / T) * (drop / soft)[:, None] + torch.exp(z) * (mark / hard)[:, None], 0.0)
    here = (p != 0) & (ids >= col_offset) & (ids < col_offset + valid)
    g.scatter_add_(1, (ids - col_offset).clamp(0, cols - 1), torch.where(here, -drop[:, None] * p, 0.0))
    if targets is not None:
        y = targets - col_offset
        here = label & (y >= 0) & (y < valid)
        g.scatter_add_(1, y.clamp(0, cols - 1)[:, None], torch.where(here, -mark, 0.0)[:, None])
    grad.copy_(g.to(logits.dtype))
    return loss, grad
