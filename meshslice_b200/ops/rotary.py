"""Rotary positions on the interleaved rows of grouped heads: per key/value head [q_0 | .. | q_group-1 | k | v] (with one query
head per key/value head the [q | k | v] rows of the attention kernels).  Native kernel for CUDA tensors, fp32 formulation for CPU
tensors."""
from __future__ import annotations

import math
from dataclasses import dataclass
from functools import cached_property
from typing import List, Optional

import torch

from .. import _native
from . import rows


@dataclass(frozen=True)
class RotaryConfig:
    """Frequencies theta^(-2 i / rot_dim) of the pairs i of the first ``rot_dim`` features of a head.

    ``layout``: 'half' pairs features (i, i + rot_dim / 2), 'interleaved' (2 i, 2 i + 1).
    ``scaling`` stretches positions to contexts ``factor`` times the trained length:
      'none'
      'linear'    every frequency divided by the factor
      'base'      theta * factor^(rot_dim / (rot_dim - 2)): the highest frequency stays, the lowest is divided by the factor
      'by_parts'  frequencies that turn more than ``beta_fast`` times over ``original_len`` positions stay, those below
                  ``beta_slow`` are divided, a linear ramp between; cosines and sines times 0.1 ln(factor) + 1
                  (``attention_factor`` in its place where given)
    """
    head_dim: int = 128
    rot_dim: int = 0                      # 0: the whole head
    theta: float = 10000.0
    layout: str = "half"
    scaling: str = "none"
    factor: float = 1.0
    original_len: int = 2048
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: Optional[float] = None

    def __post_init__(self):
        if self.rot_dim == 0:
            object.__setattr__(self, "rot_dim", self.head_dim)
        if self.head_dim <= 0 or self.head_dim % 16 or not 0 < self.rot_dim <= min(self.head_dim, 256) or self.rot_dim % 16:
            raise ValueError(f"rotary positions need multiples of 16 with 0 < rot_dim <= min(head_dim, 256) "
                             f"(got head_dim {self.head_dim}, rot_dim {self.rot_dim})")
        if self.layout not in ("half", "interleaved"):
            raise ValueError(f"unknown rotary layout {self.layout!r}")
        if self.scaling not in ("none", "linear", "base", "by_parts"):
            raise ValueError(f"unknown rotary scaling {self.scaling!r}")
        if not (self.theta > 0 and self.factor > 0 and math.isfinite(self.theta) and math.isfinite(self.factor)):
            raise ValueError("theta and factor must be positive and finite")
        if self.scaling == "by_parts" and not (self.original_len > 0 and self.beta_fast > self.beta_slow):
            raise ValueError("scaling by parts needs original_len > 0 and beta_fast > beta_slow")

    @cached_property
    def cos_factor(self) -> float:
        if self.attention_factor is not None:
            return float(self.attention_factor)
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "by_parts" else 1.0

    def frequencies(self) -> List[float]:
        """Radians per position of the pairs, in 64 bits."""
        r, s, theta = self.rot_dim, self.factor, self.theta
        if self.scaling == "base":
            theta = theta * s ** (r / (r - 2))
        f = [theta ** (-2.0 * i / r) for i in range(r // 2)]
        if self.scaling == "linear":
            f = [v / s for v in f]
        elif self.scaling == "by_parts":
            keep = [(self.original_len * v / (2 * math.pi) - self.beta_slow) / (self.beta_fast - self.beta_slow) for v in f]
            keep = [min(1.0, max(0.0, k)) for k in keep]
            f = [v * k + v / s * (1 - k) for v, k in zip(f, keep)]
        return f


class Rotary:
    """Frequencies of a ``RotaryConfig`` on a device, laid out once."""

    def __init__(self, config: RotaryConfig, device=None):
        self.config = config
        freq = config.frequencies()
        # turns per position in units of 2^-64, as two's complement
        turns = [round(math.fmod(v / (2 * math.pi), 1.0) * 2.0 ** 64) % (1 << 64) for v in freq]
        self.turns = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64, device=device)
        self._kernel = (config.head_dim, config.rot_dim, 1 if config.layout == "half" else 0)
        self._freq = torch.tensor(freq, dtype=torch.float64) if not self.turns.is_cuda else None

    def cos_sin(self, positions):
        """Cosines and sines [tokens, rot_dim / 2] in fp32 (CPU formulation)."""
        a = positions.double()[:, None] * self._freq
        return (a.cos() * self.config.cos_factor).float(), (a.sin() * self.config.cos_factor).float()


def _check(qkv, rotary: Rotary, kv_heads: int, group: int, seq, positions, out):
    width = kv_heads * (group + 2) * rotary.config.head_dim
    if kv_heads < 1 or group < 1:
        raise ValueError(f"rotary positions need kv_heads >= 1 and group >= 1 (got {kv_heads}, {group})")
    if qkv.dim() != 2 or qkv.shape[1] != width:
        raise ValueError(f"rotary positions need rows of kv_heads * (group + 2) * head_dim = {width} features (got {tuple(qkv.shape)})")
    if positions is None:
        if seq is None or seq < 1:
            raise ValueError("rotary positions need the tokens' positions or the length of a sequence")
    elif positions.dtype != torch.int64 or positions.dim() != 1 or positions.shape[0] != qkv.shape[0] or positions.device != qkv.device:
        raise ValueError(f"positions must be int64 [tokens] on the rows' device (got {positions.dtype} {tuple(positions.shape)} "
                         f"on {positions.device})")
    if out is not None and (out.shape != qkv.shape or out.dtype != qkv.dtype or out.device != qkv.device):
        raise ValueError("out must have the rows' shape, type and device")
    if rotary.turns.device != qkv.device:
        raise ValueError(f"the frequencies are on {rotary.turns.device}, the rows on {qkv.device}")


def rotary_qkv(qkv, rotary: Rotary, kv_heads: int, group: int = 1, seq: Optional[int] = None, positions=None,
               inverse: bool = False, out=None):
    """Query and key heads of ``qkv`` [tokens, kv_heads * (group + 2) * head_dim] turned to the tokens' positions, value heads as
    they are.  ``positions``: int64 [tokens]; without them token t is at t % ``seq``.  ``inverse`` turns back: the gradient of the
    unrotated rows from that of the rotated ones (times the same factor of cosines and sines).  ``out=qkv`` works in place.
    """
    c = rotary.config
    if qkv.is_cuda:
        # the common call, checked in a few steps: a kernel of 3 us is over before a longer list of them
        if out is None and qkv.dtype is torch.bfloat16 and qkv.dim() == 2 and qkv.is_contiguous() and kv_heads > 0 and group > 0:
            n, width = qkv.shape
            turns, dev, x = rotary.turns, qkv.get_device(), qkv.data_ptr()
            if positions is None:
                at, fine, length = 0, seq is not None and seq > 0, seq
            else:
                at, length = positions.data_ptr(), 1
                fine = (positions.dtype is torch.int64 and positions.dim() == 1 and positions.shape[0] == n
                        and positions.is_contiguous() and positions.get_device() == dev)
            D, rot, half = rotary._kernel
            if fine and n and x & 15 == 0 and width == kv_heads * (group + 2) * D and turns.get_device() == dev:
                stream = _native.stream_on(dev)
                y = torch.empty_like(qkv)
                _native.load().rotary(x, y.data_ptr(), width, width, at, turns.data_ptr(), n, length, kv_heads, group, D, rot, half,
                                      -1.0 if inverse else 1.0, c.cos_factor, stream)
                return y
        _check(qkv, rotary, kv_heads, group, seq, positions, out)
        if qkv.dtype != torch.bfloat16:
            raise ValueError(f"the rotary kernel needs bf16 rows (got {qkv.dtype})")
        _native.check_device(qkv)
        x = rows.as_aligned(qkv)
        if out is None or not rows.aligned(out):
            y = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device) if x is qkv else x
        else:
            y = out
            same = x.data_ptr() == y.data_ptr() and rows.pitch(x) == rows.pitch(y)
            if not same and qkv.shape[0] and rows.overlap(x, y):
                x = x.clone()
        if positions is not None and not positions.is_contiguous():
            positions = positions.contiguous()
        if qkv.shape[0]:
            _native.load().rotary(x.data_ptr(), y.data_ptr(), rows.pitch(x), rows.pitch(y),
                                  0 if positions is None else positions.data_ptr(), rotary.turns.data_ptr(), qkv.shape[0],
                                  seq if positions is None else 1, kv_heads, group, *rotary._kernel,
                                  -1.0 if inverse else 1.0, c.cos_factor, _native.stream_ptr())
        if out is not None and y is not out:
            out.copy_(y)
            return out
        return y
    _check(qkv, rotary, kv_heads, group, seq, positions, out)
    pos = torch.arange(qkv.shape[0]) % seq if positions is None else positions
    cos, sin = rotary.cos_sin(pos)
    cos, sin = cos[:, None, None], (-sin if inverse else sin)[:, None, None]
    x = qkv.float().reshape(qkv.shape[0], kv_heads, group + 2, c.head_dim)
    y, h = x.clone(), c.rot_dim // 2
    i0, i1 = (slice(0, h), slice(h, 2 * h)) if c.layout == "half" else (slice(0, 2 * h, 2), slice(1, 2 * h, 2))
    a, b = x[:, :, :-1, i0], x[:, :, :-1, i1]
    y[:, :, :-1, i0] = a * cos - b * sin
    y[:, :, :-1, i1] = b * cos + a * sin
    y = y.reshape(qkv.shape).to(qkv.dtype)
    return y if out is None else out.copy_(y)

