"""Orthogonal update of matrices by products alone: singular values to about 1, singular vectors as they are.

    X = G / |G| (Frobenius norm; 0 for G = 0),  then ``steps`` times  X <- a X + (b A + c A^2) X  with A = X X^T

of the matrix or its transpose, whichever is wider.  The default coefficients take any singular value of X above about 0.01 to 0.7 .. 1.2 in
five steps.  Native kernels for CUDA tensors, fp32 formulation for CPU tensors.

On a GPU X is held in fp32; the factors of the products are fp16 copies of X, A and b A + c A^2, and of the two symmetric products half
of the tiles are computed.  The result is about 1e-3 off the polynomial's: small singular values grow by 500 in five steps, and with
them what X was rounded by, which is why X itself is not held in 16 bits (2e-2 to 2e-1 in bf16 for matrices of falling spectra).
"""
from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional, Tuple

import torch

from .. import _native
from .gemm import _SM_COUNT, sm_count

_TYPES = (torch.float32, torch.bfloat16)
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
WORKSPACE_BYTES = 2 << 30       # matrices of a batch are taken some at a time beyond it


@lru_cache(maxsize=64)
def _check_coefficients(steps: int, coefficients: Tuple[float, float, float]):
    """The fp16 copies of X, A and b A + c A^2 are scaled for singular values of up to 4 and a polynomial of up to 200."""
    a, b, c = coefficients
    s = [i / 1000 for i in range(1001)]
    for _ in range(steps):
        if max(abs(v) for v in s) > 4 or max(abs(b * v * v + c * v ** 4) for v in s) > 200:
            raise ValueError(f"the polynomial of {coefficients} takes singular values out of range within {steps} steps")
        s = [v * (a + b * v * v + c * v ** 4) for v in s]
    if not all(math.isfinite(v) for v in s):
        raise ValueError(f"the polynomial of {coefficients} takes singular values out of range within {steps} steps")


def check_polynomial(steps, coefficients) -> Tuple[int, Tuple[float, float, float]]:
    if steps < 1 or int(steps) != steps:
        raise ValueError(f"the number of steps is positive (got {steps})")
    coefficients = tuple(coefficients)
    if len(coefficients) != 3 or not all(map(math.isfinite, coefficients)):
        raise ValueError(f"three finite coefficients (got {coefficients})")
    _check_coefficients(int(steps), coefficients)
    return int(steps), coefficients


def check_kernels(rows: int, cols: int, steps: int):
    """What the kernels take beside it."""
    if max(rows, cols) >= 1 << 24 or steps > _native.load().UNIT_STEPS:
        raise ValueError(f"the kernels take matrices of fewer than 2^24 rows and columns and at most {_native.load().UNIT_STEPS} steps "
                         f"(got {rows} x {cols}, {steps})")


def _own_elements(t) -> bool:
    """Every element has memory of its own: along each dimension a step leads beyond what the shorter steps reach."""
    reach = 0
    for step, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if step <= reach:
            return False
        reach += step * (n - 1)
    return True


def _meet(a, b) -> bool:
    """The memory of two tensors may have a byte in common, in one storage or in several over the same memory."""
    span = lambda t: (t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def orthogonalize(g, steps: int = 5, coefficients=COEFFICIENTS, out: Optional[torch.Tensor] = None, out_dtype=torch.bfloat16):
    """``g`` [rows, cols] or a batch of them [n, rows, cols], fp32 or bf16; the result, of the same shape, goes to ``out`` (fp32 or bf16, which may
    be ``g``) or a new tensor of ``out_dtype``."""
    if g.dim() not in (2, 3) or g.dtype not in _TYPES:
        raise ValueError(f"matrices are fp32 or bf16 [rows, cols] or [n, rows, cols] (got {g.dtype} {tuple(g.shape)})")
    steps, coefficients = check_polynomial(steps, coefficients)
    if out is None:
        if out_dtype not in _TYPES:
            raise ValueError(f"the result is fp32 or bf16 (got {out_dtype})")
        out = torch.empty(g.shape, dtype=out_dtype, device=g.device)
    elif out.shape != g.shape or out.dtype not in _TYPES or out.device != g.device:
        raise ValueError(f"out must be fp32 or bf16 {tuple(g.shape)} on {g.device} (got {out.dtype} {tuple(out.shape)} on {out.device})")
    elif not _own_elements(out):
        raise ValueError(f"out needs an element for each of the result's (got {tuple(out.shape)} with strides {out.stride()})")
    if g.is_cuda:
        _native.check_device(g)
    if g.numel() == 0:
        return out
    if not g.is_cuda:
        return out.copy_(_reference(g, steps, coefficients))
    batch, target = (g[None], out[None]) if g.dim() == 2 else (g, out)
    items, r, c = batch.shape
    check_kernels(r, c, steps)
    if not batch[0].is_contiguous():
        batch = batch.contiguous()
    if out is not g and _meet(batch, target):       # a matrix is read before its own result is written, not before those of others
        batch = batch.clone()
    result = target
    if min(target.stride(1), target.stride(2)) != 1 or (r > 1 and c > 1 and target.stride(1) == target.stride(2)):
        result = torch.empty(target.shape, dtype=target.dtype, device=target.device)
    m, n = -(-min(r, c) // 64) * 64, -(-max(r, c) // 64) * 64
    C, sms, status, stream = _native.load(), _SM_COUNT.get(g.get_device()) or sm_count(g.device), _native.status().dev, _native.stream_ptr()
    if r <= C.UNIT_SIDE and c <= C.UNIT_SIDE:      # in one launch, without a workspace
        most, space = items, 0
    else:
        each = C.unit_space(m, n)
        most = max(1, min(items, WORKSPACE_BYTES // each, (1 << 31) // m - 1))
        block = torch.empty(most * each, dtype=torch.uint8, device=g.device)
        space = block.data_ptr()
    stride, strides = batch.stride(0) if items > 1 else 0, (result.stride(0) if items > 1 else 0, result.stride(1), result.stride(2))
    for i in range(0, items, most):
        C.orthogonalize(batch.data_ptr() + i * stride * batch.element_size(), 1 if batch.dtype is torch.bfloat16 else 0, stride,
                        min(most, items - i), r, c, steps, *coefficients, space, m, n,
                        result.data_ptr() + i * strides[0] * result.element_size(), 1 if result.dtype is torch.float32 else 0, *strides, sms,
                        status, stream)
    if result is not target:
        target.copy_(result)
    return out


def _reference(g, steps: int, coefficients):
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = torch.where(norm == 0, 0.0, x.double() / norm).float()
    a, b, c = coefficients
    for _ in range(steps):
        q = x @ x.mT
        x = a * x + (b * q + c * (q @ q)) @ x
    return x.mT if tall else x
