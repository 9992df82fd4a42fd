"""AdamW with fp32 master weights over the flat parameter buffers of a rank.

bf16 parameters are what the forward pass reads; the optimizer keeps fp32 master copies and
moments, reads bf16 (sharded weights) or fp32 (row-replicated parameters) gradients, and writes
both the master and the bf16 copy in one fused kernel per buffer.  Gradient clipping uses the
global L2 norm: sharded parameters contribute once per rank, row-replicated parameters once per
mesh column.
"""
from __future__ import annotations

import math
from typing import List, Optional

import torch

from . import _native
from .ops.orthogonal import COEFFICIENTS, check_kernels, check_polynomial, orthogonalize


class FlatGroup:
    """One contiguous parameter buffer with its gradient buffer (same element count)."""

    def __init__(self, param: torch.Tensor, grad: torch.Tensor, kind: str):
        assert param.numel() == grad.numel() and param.numel() % 4 == 0
        self.param, self.grad, self.kind = param, grad, kind
        self.master = param.float().clone()
        self.m = torch.zeros_like(self.master)
        self.v = torch.zeros_like(self.master)


def _check_buffers(param, grad):
    """What the kernels read and write of a group, four elements at a time."""
    if param.dtype != torch.bfloat16 or grad.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"the optimizer's kernels need bf16 parameters with fp32 or bf16 gradients (got {param.dtype}, {grad.dtype})")
    for t in (param, grad):
        if not t.is_contiguous() or t.data_ptr() % (4 * t.element_size()):
            raise ValueError("the optimizer's kernels need contiguous buffers that begin on a boundary of four elements")


class AdamW:
    def __init__(self, groups: List[FlatGroup], lr: float = 1e-4, betas=(0.9, 0.95), eps: float = 1e-8,
                 weight_decay: float = 0.0, max_grad_norm: Optional[float] = 1.0, mesh=None):
        for g in groups:
            if g.param.is_cuda:
                _check_buffers(g.param, g.grad)
        self.groups, self.lr, self.betas, self.eps, self.wd = groups, lr, betas, eps, weight_decay
        self.max_grad_norm, self.mesh = max_grad_norm, mesh
        self.step_count = 0
        dev = groups[0].param.device
        self._sq = torch.zeros(2, dtype=torch.float32, device=dev)
        self._scale = torch.ones(1, dtype=torch.float32, device=dev)
        self.last_grad_norm = None

    def _grad_scale(self):
        """Device scalar that rescales the gradients so that their global norm is <= max."""
        if self.max_grad_norm is None:
            return None
        _native.zero_(self._sq)
        for g in self.groups:
            idx = 0 if g.kind == "sharded" else 1
            if g.grad.is_cuda:
                _native.load().sumsq(g.grad.data_ptr(), 1 if g.grad.dtype == torch.float32 else 0,
                                     g.grad.numel(), self._sq[idx:idx + 1].data_ptr(), _native.stream_ptr())
            else:
                self._sq[idx] += g.grad.float().pow(2).sum()
        sq = self._sq
        if self.mesh is not None and self.mesh.R * self.mesh.C > 1 and hasattr(self.mesh, "dist"):
            d = self.mesh.dist
            sq = sq.clone()
            if self.mesh.R > 1:
                # replicated parameters are identical along a mesh column: count them once
                sq[1] = sq[1] / self.mesh.R
            d.all_reduce(sq, group=self.mesh.group)
        if sq.is_cuda:
            norm = torch.empty((), dtype=torch.float32, device=sq.device)
            _native.load().clip_scale(sq.data_ptr(), sq.numel(), self.max_grad_norm, norm.data_ptr(),
                                      self._scale.data_ptr(), _native.stream_ptr())
        else:
            norm = torch.sqrt(sq.sum())
            self._scale.copy_(torch.clamp(self.max_grad_norm / (norm + 1e-6), max=1.0).reshape(1))
        self.last_grad_norm = norm
        return self._scale

    def step(self):
        self._step()

    def _step(self):
        """AdamW on the spans of the groups; returns the gradients' scale."""
        self.step_count += 1
        b1, b2 = self.betas
        bc1, bc2 = 1 - b1 ** self.step_count, 1 - b2 ** self.step_count
        scale = self._grad_scale()
        for g in self.groups:
            for a, b in self._spans(g):
                param, grad, master, m, v = g.param, g.grad, g.master, g.m, g.v
                if b - a != param.numel():
                    param, grad, master, m, v = (t[a:b] for t in (param, grad, master, m, v))
                if param.is_cuda:
                    _native.load().adamw_step(param.data_ptr(), master.data_ptr(), m.data_ptr(), v.data_ptr(),
                                              grad.data_ptr(), 1 if grad.dtype == torch.float32 else 0,
                                              param.numel(), self.lr, b1, b2, self.eps, self.wd, bc1, bc2,
                                              0 if scale is None else scale.data_ptr(), _native.stream_ptr())
                else:
                    gr = grad.float() * (1.0 if scale is None else scale.item())
                    m.mul_(b1).add_(gr, alpha=1 - b1)
                    v.mul_(b2).addcmul_(gr, gr, value=1 - b2)
                    upd = (m / bc1) / ((v / bc2).sqrt() + self.eps) + self.wd * master
                    master.add_(upd, alpha=-self.lr)
                    param.copy_(master.to(param.dtype))
        return scale

    def _spans(self, g: FlatGroup):
        """The elements of a group that this step updates, as (first, end) pairs."""
        return [(0, g.param.numel())]

    def zero_grad(self):
        for g in self.groups:
            _native.zero_(g.grad)

    def resync_from_params(self, step: int = 0):
        """Rebuild the optimizer state from the current bf16 parameters: the fp32 master copies
        become the parameters, both moments are cleared and the step counter is set.  Needed after
        parameters were written behind the optimizer's back (a checkpoint without optimizer
        state, imported weights); otherwise the next step would overwrite them from the stale
        master copies."""
        self.step_count = int(step)
        for g in self.groups:
            g.master.copy_(g.param.float())
            g.m.zero_()
            g.v.zero_()

    def named_state(self, params):
        """Views of the flat master / m / v buffers per named parameter shard.

        ``params`` is ``model.parameters()``.  Returns {name: {coord: (master, m, v)}} where each
        view has the shape of the parameter shard; a parameter that does not live inside one of
        this optimizer's flat buffers is an error.  This is what makes the optimizer state
        save-able and re-shardable with the same rules as the parameters themselves."""
        out = {name: {} for name, _, _, _ in params}
        for name, key, t, g, off in self._located(params):
            out[name][key] = tuple(b[off:off + t.numel()].view(t.shape) for b in (g.master, g.m, g.v))
        return out

    def _located(self, params):
        """(name, coordinate, shard, group, its first element there) of every parameter shard."""
        spans = [(g, g.param.data_ptr(), g.param.data_ptr() + g.param.numel() * g.param.element_size())
                 for g in self.groups]
        for name, p, _, _ in params:
            for key, t in p.shards.items():
                for g, lo, hi in spans:
                    if lo <= t.data_ptr() < hi:
                        if not t.is_contiguous():
                            raise ValueError(f"{name}: parameter shard is not contiguous in its flat buffer")
                        yield name, key, t, g, (t.data_ptr() - lo) // g.param.element_size()
                        break
                else:
                    raise ValueError(f"{name}: parameter shard {key} is outside the optimizer's flat buffers")

    def update_rules(self, params):
        """{name: 'adamw', 'orthogonal' or 'both'}: what updates a parameter, and so what its m and v mean."""
        out = {}
        for name, _, t, g, off in self._located(params):
            here = sum(max(0, min(b, off + t.numel()) - max(a, off)) for a, b in self._spans(g))
            out[name] = "adamw" if here == t.numel() else "orthogonal" if here == 0 else "both"
        return out

    def state_dict(self):
        return {"step": self.step_count,
                "groups": [{"master": g.master, "m": g.m, "v": g.v, "kind": g.kind, "adamw": self._spans(g)} for g in self.groups]}

    def load_state_dict(self, sd):
        for i, (g, s) in enumerate(zip(self.groups, sd["groups"])):
            own, at = self._spans(g), 0
            if "adamw" in s:
                same = [tuple(x) for x in s["adamw"]] == own
            else:
                same = True
                for a, b in own + [(g.param.numel(), g.param.numel())]:
                    same &= found_rule(s["m"][at:a], s["v"][at:a]) in (None, "orthogonal")
                    same &= found_rule(s["m"][a:b], s["v"][a:b]) in (None, "adamw")
                    at = b
            if not same:
                raise ValueError(f"group {i}: {OTHER_RULE}")
        self.step_count = sd["step"]
        for g, s in zip(self.groups, sd["groups"]):
            g.master.copy_(s["master"])
            g.m.copy_(s["m"])
            g.v.copy_(s["v"])
            g.param.copy_(g.master.to(g.param.dtype))


OTHER_RULE = ("the moments are those of another optimizer (AdamW's are means, those of orthogonal updates an undamped sum beside no second one); "
              "without them the parameters can be loaded alone, and resync_from_params starts the optimizer anew")


def found_rule(m, v) -> Optional[str]:
    """The update rule of a state that does not name it: orthogonal updates leave v at 0, AdamW does not beside a first moment of this
    size, whose square is far above the smallest fp32 number.  None: nothing that tells."""
    orthogonal, adamw = bool(((m.abs() > 1e-12) & (v == 0)).any()), bool(v.any())
    return "both" if orthogonal and adamw else "orthogonal" if orthogonal else "adamw" if adamw else None


UPDATE_BYTES = 1 << 30      # of updates that are in memory at a time


class Muon(AdamW):
    """Orthogonal updates of matrices, AdamW for everything else in the flat buffers.  Per matrix, with its gradient g (clipped by the norm of
    all gradients):

        m <- momentum m + g        u = g + momentum m (nesterov) or m
        w <- w - lr (0.2 sqrt(max(rows, columns)) orthogonalize(u) + weight_decay w)

    whose elements are of the size of AdamW's, so that one learning rate serves both.  ``matrices``: whole 2-D views of the groups'
    parameters; those of one shape that lie at equal distances are updated together.  Their m is kept in the group's first
    moment, and the second one stays 0: a state saved by one of the two optimizers is refused by the other.
    """

    def __init__(self, groups: List[FlatGroup], matrices: List[torch.Tensor], momentum: float = 0.95, nesterov: bool = True, steps: int = 5,
                 coefficients=COEFFICIENTS, **kw):
        super().__init__(groups, **kw)
        if self.mesh is not None and self.mesh.R * self.mesh.C > 1:
            raise ValueError("orthogonal updates are of whole matrices: a 1 x 1 mesh")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"momentum must be in [0, 1) (got {momentum})")
        self.momentum, self.nesterov = momentum, nesterov
        self.steps, self.coefficients = check_polynomial(steps, coefficients)
        self._stacks = []                 # (group, first element, distance, count, rows, columns)
        self._rest = {}                   # of the groups, by identity of the group: spans that AdamW updates
        taken = {id(g): [] for g in groups}
        found = sorted((self._place(w) + tuple(w.shape) for w in matrices), key=lambda t: (t[0], t[2:], t[1]))
        for k, at, r, c in found:
            taken[id(groups[k])].append((at, at + r * c))
            last = self._stacks[-1] if self._stacks else None
            if last is not None and (last[0], *last[4:]) == (k, r, c):
                first, gap, n = last[1:4]
                if (n == 1 and at >= first + r * c) or (n > 1 and at == first + n * gap):
                    self._stacks[-1] = (k, first, at - first if n == 1 else gap, n + 1, r, c)
                    continue
            self._stacks.append((k, at, r * c, 1, r, c))
        for g in groups:
            at, rest = 0, []
            for a, b in sorted(taken[id(g)]) + [(g.param.numel(), g.param.numel())]:
                if a < at:
                    raise ValueError("two of the matrices share elements")
                if a > at:
                    rest.append((at, a))
                at = b
            self._rest[id(g)] = rest

    def _place(self, w: torch.Tensor):
        if w.dim() != 2 or not w.is_contiguous() or w.numel() % 4 or w.numel() == 0:
            raise ValueError(f"matrices are contiguous, of a multiple of 4 elements, and not empty (got {tuple(w.shape)})")
        if w.is_cuda:
            check_kernels(*w.shape, self.steps)
        for k, g in enumerate(self.groups):
            at = w.data_ptr() - g.param.data_ptr()
            if w.dtype == g.param.dtype and 0 <= at < g.param.numel() * g.param.element_size():
                at //= g.param.element_size()
                if at % 4 or at + w.numel() > g.param.numel():
                    raise ValueError("a matrix begins at a multiple of 4 elements of its flat buffer and ends in it")
                return k, at
        raise ValueError("a matrix lies outside the optimizer's flat buffers")

    def _spans(self, g: FlatGroup):
        return self._rest[id(g)]

    def step(self):
        scale = self._step()
        for k, first, gap, count, r, c in self._stacks:
            some = max(1, min(count, UPDATE_BYTES // (4 * r * c)))
            for i in range(0, count, some):
                self._update(k, first + i * gap, gap, min(some, count - i), r, c, scale)

    def _update(self, k: int, at: int, gap: int, n: int, r: int, c: int, scale):
        """``n`` matrices of group ``k``, ``gap`` elements apart from element ``at`` on."""
        g, size = self.groups[k], 0.2 * math.sqrt(max(r, c))
        if g.param.is_cuda:
            _native.check_device(g.param)
            C, stream = _native.load(), _native.stream_ptr()
            u = torch.empty(n, r, c, dtype=torch.float32, device=g.param.device)
            wide = g.grad.element_size()
            C.momentum_step(g.grad.data_ptr() + at * wide, 1 if wide == 4 else 0, g.m.data_ptr() + at * 4, u.data_ptr(), n, r * c, gap,
                            self.momentum, 1 if self.nesterov else 0, 0 if scale is None else scale.data_ptr(), stream)
            orthogonalize(u, self.steps, self.coefficients, out=u)
            C.apply_update(u.data_ptr(), g.master.data_ptr() + at * 4, g.param.data_ptr() + at * g.param.element_size(), n, r * c, gap,
                           self.lr, size, self.wd, stream)
            return
        view = lambda t: t.as_strided((n, r, c), (gap, c, 1), t.storage_offset() + at)
        grad = view(g.grad).float() * (1.0 if scale is None else scale.item())
        m, master = view(g.m), view(g.master)
        m.mul_(self.momentum).add_(grad)
        u = grad + self.momentum * m if self.nesterov else m
        master.sub_(self.lr * (size * orthogonalize(u, self.steps, self.coefficients, out_dtype=torch.float32) + self.wd * master))
        view(g.param).copy_(master.to(g.param.dtype))
