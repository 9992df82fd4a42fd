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
from .gemm import sm_count

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
WORKSPACE_BYTES = 2 << 30       # matrices of a batch are taken some at a time beyond it
# powers of two that the fp16 copies are scaled by: their largest values are below 4, 16 and 255 (what the coefficients are checked for)
_SX, _SA, _SB = 2.0 ** 10, 2.0 ** 10, 2.0 ** 8


@lru_cache(maxsize=64)
def _check_coefficients(steps: int, coefficients: Tuple[float, float, float]):
    a, b, c = coefficients
    s = [i / 1000 for i in range(1001)]
    for _ in range(steps):
        if max(abs(v) for v in s) > 4 or max(abs(b * v * v + c * v ** 4) for v in s) > 200:
            raise ValueError(f"the polynomial of {coefficients} takes singular values out of range within {steps} steps")
        s = [v * (a + b * v * v + c * v ** 4) for v in s]
    if not all(math.isfinite(v) for v in s):
        raise ValueError(f"the polynomial of {coefficients} takes singular values out of range within {steps} steps")


def orthogonalize(g, steps: int = 5, coefficients=COEFFICIENTS, out: Optional[torch.Tensor] = None, out_dtype=torch.bfloat16):
    """``g`` [rows, cols] or a batch of them [n, rows, cols], fp32 or bf16; the result, of the same shape, goes to ``out`` (fp32 or bf16, which may
    be ``g``) or a new tensor of ``out_dtype``."""
    if g.dim() not in (2, 3) or g.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"matrices are fp32 or bf16 [rows, cols] or [n, rows, cols] (got {g.dtype} {tuple(g.shape)})")
    if steps < 1 or int(steps) != steps:
        raise ValueError(f"the number of steps is positive (got {steps})")
    coefficients = tuple(float(v) for v in coefficients)
    if len(coefficients) != 3 or not all(math.isfinite(v) for v in coefficients):
        raise ValueError(f"three finite coefficients (got {coefficients})")
    _check_coefficients(int(steps), coefficients)
    if out is None:
        if out_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"the result is fp32 or bf16 (got {out_dtype})")
        out = torch.empty(g.shape, dtype=out_dtype, device=g.device)
    elif out.shape != g.shape or out.dtype not in (torch.float32, torch.bfloat16) or out.device != g.device:
        raise ValueError(f"out must be fp32 or bf16 {tuple(g.shape)} on {g.device} (got {out.dtype} {tuple(out.shape)} on {out.device})")
    if g.is_cuda:
        _native.check_device(g)
    if g.numel() == 0:
        return out
    if not g.is_cuda:
        return out.copy_(_reference(g, int(steps), coefficients))
    batch, target = (g[None], out[None]) if g.dim() == 2 else (g, out)
    items, r, c = batch.shape
    if max(r, c) >= 1 << 24:
        raise ValueError(f"the kernels take matrices of fewer than 2^24 rows and columns (got {r} x {c})")
    if not batch[0].is_contiguous():
        batch = batch.contiguous()
    result = target
    if min(target.stride(1), target.stride(2)) != 1 or (r > 1 and c > 1 and target.stride(1) == target.stride(2)):
        result = torch.empty(target.shape, dtype=target.dtype, device=target.device)
    m, n = -(-min(r, c) // 64) * 64, -(-max(r, c) // 64) * 64
    each = 8 * m * n + 4 * m * m + 8 * _native.load().NORM_PARTS
    most = int(max(1, min(items, WORKSPACE_BYTES // each, (1 << 31) // m - 1)))
    space = torch.empty(most * each, dtype=torch.uint8, device=g.device)
    for i in range(0, items, most):
        _some(batch[i:i + most], result[i:i + most], int(steps), coefficients, m, n, space)
    return out if result is target else _copied(out, target, result)


def _copied(out, target, result):
    target.copy_(result)
    return out


def _some(g, out, steps: int, coefficients, m: int, n: int, space):
    C, sms, status, stream = _native.load(), sm_count(g.device), _native.status().dev, _native.stream_ptr()
    items, r, c = g.shape
    tall = r > c
    a, b, cc = coefficients
    at = space.data_ptr()
    x, xs, ys = at, at + 4 * items * m * n, at + 6 * items * m * n
    q, p = at + 8 * items * m * n, at + 8 * items * m * n + 2 * items * m * m
    norms = at + 8 * items * m * n + 4 * items * m * m
    C.unit_load(g.data_ptr(), 1 if g.dtype == torch.bfloat16 else 0, g.stride(0) if items > 1 else 0, items, r, c, 1 if tall else 0, norms, x, xs,
                m, n, _SX, stream)
    s_row, s_col = (out.stride(2), out.stride(1)) if tall else (out.stride(1), out.stride(2))
    for k in range(steps):
        last = k == steps - 1
        C.gram(items, m, n, xs, q, 0, _SA / _SX ** 2, 0.0, sms, status, stream)
        C.gram(items, m, m, q, p, q, _SB * cc / _SA ** 2, _SB * b / _SA, sms, status, stream)
        C.ortho_step(items, m, n, p, xs, x, ys, _SX, a, 1 / (_SB * _SX), out.data_ptr() if last else 0, min(r, c), max(r, c),
                     out.stride(0) if items > 1 else 0, s_row, s_col, 1 if out.dtype == torch.float32 else 0, sms, status, stream)
        xs, ys = ys, xs


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
