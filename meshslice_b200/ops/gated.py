"""Gated feed-forward block  y = (act(x Wg) * (x Wu)) Wd  with its gradients.  Native kernels for CUDA tensors, fp32 formulation for
CPU tensors.

act is 'silu' (x sigmoid(x)) or 'gelu' (tanh form).  Gate and up weights lie as [inputs, features] (layout 'nn') or [features, inputs]
('nt'), the down weight as [features, outputs] ('nn') or [outputs, features] ('nt').

    dh = dy Wd^T     du = dh act(g)     dg = dh u act'(g)        g = x Wg, u = x Wu, h = act(g) u
    dWd = h^T dy     dWg = x^T dg       dWu = x^T du             dx = dg Wg^T + du Wu^T

On a GPU both projections, the activation and the product are one kernel; what it keeps of g and u for the gradient has 11 significant
bits, in a range that 32 features of a token share.  h, dg and du are rounded to bf16, as inputs of products are.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from .. import _native
from . import rows
from .gemm import _SM_COUNT, sm_count

ACTS = {"silu": 0, "gelu": 1}
_LAYOUTS = ("nn", "nt")
_BF16, _F32 = torch.bfloat16, torch.float32


@dataclass
class GatedSaved:
    """What a forward pass keeps for the backward one: h, gate and up.  On a GPU in one block of bytes: h (bf16), gate and up (fp16 beside an
    exponent for 32 features), the exponents."""
    tokens: int
    features: int
    device: torch.device
    block: Optional[torch.Tensor] = None
    h: Optional[torch.Tensor] = None
    gate: Optional[torch.Tensor] = None
    up: Optional[torch.Tensor] = None


def _at(t, pitch: int):
    """(tensor, address, row pitch) as the kernels take a matrix whose rows are ``pitch`` long; a copy where they cannot address it."""
    if t.is_contiguous():
        p = t.data_ptr()
        if p & 15 == 0:
            return t, p, pitch
    t = rows.as_aligned(t)
    return t, t.data_ptr(), rows.pitch(t)


def _sizes(x, w_gate, w_up, w_down, act: str, up_layout: str, down_layout: str) -> Tuple[int, int, int, int]:
    """(tokens, inputs, features, outputs) after all checks that do not depend on the direction."""
    if act not in ACTS:
        raise ValueError(f"unknown activation {act!r}: one of {sorted(ACTS)}")
    if up_layout not in _LAYOUTS or down_layout not in _LAYOUTS:
        raise ValueError(f"weights lie as 'nn' or 'nt' (got {up_layout!r}, {down_layout!r})")
    if any(t.dim() != 2 for t in (x, w_gate, w_up, w_down)):
        raise ValueError("x and the weights are matrices")
    n, d = x.shape
    i, f = w_gate.shape if up_layout == "nn" else w_gate.shape[::-1]
    j, o = w_down.shape if down_layout == "nn" else w_down.shape[::-1]
    if w_up.shape != w_gate.shape or i != d or j != f:
        raise ValueError(f"shapes do not fit: x {tuple(x.shape)}, gate {tuple(w_gate.shape)}, up {tuple(w_up.shape)} ({up_layout}), "
                         f"down {tuple(w_down.shape)} ({down_layout})")
    if d < 1 or f < 1 or o < 1:
        raise ValueError(f"inputs, features and outputs must not be empty (got {d}, {f}, {o})")
    dtype, at = x.dtype, x.get_device()
    for t in (w_gate, w_up, w_down):
        if t.dtype is not dtype or t.get_device() != at:
            raise ValueError(f"x is {x.dtype} on {x.device}, a weight {t.dtype} on {t.device}")
    if x.is_cuda:
        if dtype is not _BF16:
            raise ValueError(f"the gated kernels need bf16 (got {x.dtype})")
        if d % 8 or f % 8 or o % 8:
            raise ValueError(f"the gated kernels need multiples of 8 features (got {d}, {f}, {o})")
        if n >= 1 << 31:
            raise ValueError(f"the gated kernels take fewer than 2^31 tokens (got {n})")
        _native.check_device(x)
    return n, d, f, o


def gated_ff_fwd(x, w_gate, w_up, w_down, act: str = "silu", up_layout: str = "nn", down_layout: str = "nn", keep: bool = True):
    """(y [tokens, outputs], what ``gated_ff_bwd`` needs, None without ``keep``)."""
    n, d, f, o = _sizes(x, w_gate, w_up, w_down, act, up_layout, down_layout)
    if not x.is_cuda:
        xf = x.float()
        g, u = (xf @ (w.float() if up_layout == "nn" else w.float().T) for w in (w_gate, w_up))
        h = _act(g, act)[0] * u
        y = h @ (w_down.float() if down_layout == "nn" else w_down.float().T)
        return y.to(x.dtype), GatedSaved(n, f, x.device, h=h, gate=g, up=u) if keep else None
    C = _native.load()
    y = x.new_empty(n, o)
    part = n * f
    block = x.new_empty(3 * part + n * -(-f // C.GATED_CHUNK) if keep else part)
    saved = GatedSaved(n, f, x.device, block) if keep else None
    if n == 0:
        return y, saved
    up_nt, down_nt = up_layout == "nt", down_layout == "nt"
    x, px, lx = _at(x, d)
    w_gate, pg, lg = _at(w_gate, d if up_nt else f)
    w_up, pu, lu = _at(w_up, d if up_nt else f)
    w_down, pd, ld = _at(w_down, f if down_nt else o)
    at, part = block.data_ptr(), 2 * part
    C.gated_fwd(n, d, f, o, px, lx, pg, lg, pu, lu, 1 if up_nt else 0, pd, ld, 1 if down_nt else 0, y.data_ptr(), at, at + part, at + 2 * part,
                at + 3 * part, ACTS[act], 1 if keep else 0, _SM_COUNT.get(x.get_device()) or sm_count(x.device), _native.status().dev,
                _native.stream_ptr())
    return y, saved


def gated_ff_bwd(dy, x, w_gate, w_up, w_down, saved: GatedSaved, act: str = "silu", up_layout: str = "nn", down_layout: str = "nn",
                 grads: Optional[Sequence[torch.Tensor]] = None):
    """(dx, (gradients of gate, up and down weight)).  The weights' gradients are new tensors, or are added to ``grads`` (fp32 or the
    weights' type, in the weights' layouts), which share no memory with one another or with an operand; columns of one wider matrix are fine."""
    n, d, f, o = _sizes(x, w_gate, w_up, w_down, act, up_layout, down_layout)
    if dy.shape != (n, o) or dy.dtype is not x.dtype or dy.get_device() != x.get_device():
        raise ValueError(f"dy must be {x.dtype} [{n}, {o}] on {x.device} (got {dy.dtype} {tuple(dy.shape)} on {dy.device})")
    if saved is None or (saved.tokens, saved.features, saved.device) != (n, f, x.device):
        raise ValueError("the backward pass needs what the forward pass kept")
    weights = (w_gate, w_up, w_down)
    add = grads is not None
    if add:
        if len(grads) != 3:
            raise ValueError("grads are those of gate, up and down weight")
        for g, w in zip(grads, weights):
            if g.shape != w.shape or g.device != w.device or g.dtype not in (_F32, w.dtype):
                raise ValueError(f"a gradient must be fp32 or {w.dtype} {tuple(w.shape)} on {w.device} (got {g.dtype} {tuple(g.shape)} on {g.device})")
            if x.is_cuda and not rows.adds(g):
                raise ValueError("gradients that are added to need neighbouring columns and rows on 16-byte boundaries")
        rows.check_apart(grads, (dy, x, *weights), "a gradient")        # products of one launch add to them and read the operands
    if not x.is_cuda:
        g, u, xf, dyf = saved.gate, saved.up, x.float(), dy.float()
        a, da = _act(g, act)
        dh = dyf @ (w_down.float().T if down_layout == "nn" else w_down.float())
        dg, du, h = dh * (u * da), dh * a, saved.h
        back = lambda t, w: t @ (w.float().T if up_layout == "nn" else w.float())
        dx = (back(dg, w_gate) + back(du, w_up)).to(x.dtype)
        new = [xf.T @ dg, xf.T @ du] if up_layout == "nn" else [dg.T @ xf, du.T @ xf]
        new.append(h.T @ dyf if down_layout == "nn" else dyf.T @ h)
        if not add:
            return dx, tuple(t.to(x.dtype) for t in new)
        for t, v in zip(grads, new):
            t += v.to(t.dtype)
        return dx, tuple(grads)
    dx = x.new_empty(n, d)
    if not add:
        grads = (x.new_empty(w_gate.shape), x.new_empty(w_up.shape), x.new_empty(w_down.shape))
    if n == 0:
        if not add:
            for t in grads:
                t.zero_()
        return dx, tuple(grads)
    up_nt, down_nt = up_layout == "nt", down_layout == "nt"
    dy, py, ly = _at(dy, o)
    x, px, lx = _at(x, d)
    w_gate, pg, lg = _at(w_gate, d if up_nt else f)
    w_up, pu, lu = _at(w_up, d if up_nt else f)
    w_down, pd, ld = _at(w_down, f if down_nt else o)
    gg, gu, gd = grads
    if add:
        lgg, lgu, lgd = rows.pitch(gg), rows.pitch(gu), rows.pitch(gd)
        types = sum(1 << i for i, g in enumerate(grads) if g.dtype is _F32)
    else:
        lgg = lgu = d if up_nt else f
        lgd, types = f if down_nt else o, 0
    space = x.new_empty(2 * n * f)                        # dg, du
    part, at, to = 2 * n * f, saved.block.data_ptr(), space.data_ptr()
    _native.load().gated_bwd(n, d, f, o, py, ly, px, lx, pg, lg, pu, lu, 1 if up_nt else 0, pd, ld, 1 if down_nt else 0, at, at + part,
                             at + 2 * part, at + 3 * part, to, to + part, dx.data_ptr(), gg.data_ptr(), lgg, gu.data_ptr(), lgu, gd.data_ptr(), lgd,
                             types, 1 if add else 0, ACTS[act], _SM_COUNT.get(x.get_device()) or sm_count(x.device), _native.status().dev,
                             _native.stream_ptr())
    return dx, grads if type(grads) is tuple else tuple(grads)


def _same(act: str, *tensors):
    first = tensors[0]
    if act not in ACTS:
        raise ValueError(f"unknown activation {act!r}: one of {sorted(ACTS)}")
    for t in tensors[1:]:
        if t.shape != first.shape or t.dtype != first.dtype or t.device != first.device:
            raise ValueError(f"operands of one shape, type and device (got {first.dtype} {tuple(first.shape)} on {first.device}, "
                             f"{t.dtype} {tuple(t.shape)} on {t.device})")
    if first.is_cuda:
        if first.dtype != torch.bfloat16 or first.numel() % 8:
            raise ValueError(f"the gated kernels need bf16 and a multiple of 8 elements (got {first.dtype} {tuple(first.shape)})")
        _native.check_device(first)


def _block(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def gated_act(gate, up, act: str = "silu"):
    """act(gate) * up of projections that are there already."""
    _same(act, gate, up)
    if not gate.is_cuda:
        return (_act(gate.float(), act)[0] * up.float()).to(gate.dtype)
    h = torch.empty(gate.shape, dtype=gate.dtype, device=gate.device)
    if gate.numel():
        gate, up = _block(gate), _block(up)
        _native.load().gated_act(gate.data_ptr(), up.data_ptr(), h.data_ptr(), h.numel(), ACTS[act], _native.stream_ptr())
    return h


def gated_act_bwd(dh, gate, up, act: str = "silu"):
    """Gradients of ``gated_act`` for gate and up."""
    _same(act, dh, gate, up)
    if not dh.is_cuda:
        a, da = _act(gate.float(), act)
        return (dh.float() * (up.float() * da)).to(dh.dtype), (dh.float() * a).to(dh.dtype)
    dg, du = (torch.empty(dh.shape, dtype=dh.dtype, device=dh.device) for _ in range(2))
    if dh.numel():
        dh, gate, up = _block(dh), _block(gate), _block(up)
        _native.load().gated_act_bwd(dh.data_ptr(), gate.data_ptr(), up.data_ptr(), dg.data_ptr(), du.data_ptr(), dg.numel(), ACTS[act],
                                     _native.stream_ptr())
    return dg, du


def _act(g, act: str):
    """Activation and derivative in g's precision: both activations are g sigmoid(q(g)), whose small values a tanh would lose."""
    if act == "silu":
        q, dq = g, 1.0
    else:
        c, near = 2 * math.sqrt(2 / math.pi), g.clamp(-64, 64)      # beyond, s (1 - s) is 0, and g g may leave the precision's range
        q, dq = c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * near * near)
    s = torch.sigmoid(q)
    return g * s, s + g * s * (1 - s) * dq
