"""Causal attention within a window that keeps the first tokens visible, on rows of grouped heads (per key/value head
[q_0 | .. | q_group-1 | k | v]): query i sees key j <= i where i - j < window or j < sinks.  Native kernels for CUDA tensors, fp32
formulation for CPU tensors."""
from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional

import torch

from .. import _native
from . import rows

HEAD_DIM = 128          # of the kernels


def _width(qkv, kv_heads: int, group: int, batch_rows: Optional[int]) -> int:
    """Features per head of ``qkv`` [batch_rows, kv_heads * (group + 2) * D]."""
    if kv_heads < 1 or group < 1:
        raise ValueError(f"attention needs kv_heads >= 1 and group >= 1 (got {kv_heads}, {group})")
    per = kv_heads * (group + 2)
    if qkv.dim() != 2 or qkv.shape[1] % per or qkv.shape[1] == 0 or (batch_rows is not None and qkv.shape[0] != batch_rows):
        raise ValueError(f"attention needs rows [{'tokens' if batch_rows is None else batch_rows}, kv_heads * (group + 2) * head_dim] with "
                         f"kv_heads * (group + 2) = {per} (got {tuple(qkv.shape)})")
    return qkv.shape[1] // per


# ----------------------------------------------------------------------------------------------
# whole sequences
# ----------------------------------------------------------------------------------------------
@lru_cache(maxsize=256)
def _scratch(batch: int, seq: int, kv_heads: int, group: int, window: int, sinks: int) -> int:
    return _native.load().window_attention_scratch(batch, seq, kv_heads, group, window, sinks)


_SCALE = 1.0 / math.sqrt(HEAD_DIM)


def _check(qkv, batch: int, seq: int, kv_heads: int, group: int, window: int, sinks: int) -> int:
    if (qkv.is_cuda and qkv.dtype is torch.bfloat16 and batch >= 0 and seq > 0 and kv_heads > 0 and group > 0 and window >= 0 and sinks >= 0
            and qkv.shape == (batch * seq, kv_heads * (group + 2) * HEAD_DIM)):
        return HEAD_DIM
    if batch < 0 or seq < 1 or window < 0 or sinks < 0:
        raise ValueError(f"attention needs seq >= 1, window >= 0 (0: no window) and sinks >= 0 (got batch {batch}, seq {seq}, "
                         f"window {window}, sinks {sinks})")
    D = _width(qkv, kv_heads, group, batch * seq)
    if qkv.is_cuda:
        if qkv.dtype != torch.bfloat16 or D != HEAD_DIM:
            raise ValueError(f"the window attention kernel needs bf16 rows with head_dim {HEAD_DIM} (got {qkv.dtype}, {D})")
    return D


def _dense(t):
    """``t`` as one block of memory on a 16-byte boundary: the kernels address whole rows without a pitch."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _formulation(qkv, batch, seq, kv_heads, group, window, sinks, D):
    """fp32 q [b, kv, g, s, D], k and v [b, kv, 1, s, D] and the masked scores."""
    x = qkv.float().view(batch, seq, kv_heads, group + 2, D).permute(0, 2, 3, 1, 4)
    q, k, v = x[:, :, :group], x[:, :, group:group + 1], x[:, :, group + 1:]
    i, j = torch.arange(seq)[:, None], torch.arange(seq)[None, :]
    hidden = (j > i) | ((i - j >= (window or seq)) & (j >= sinks))
    return q, k, v, (q @ k.transpose(-1, -2) / math.sqrt(D)).masked_fill(hidden, -math.inf)


def window_attention_fwd(qkv, batch: int, seq: int, kv_heads: int, group: int = 1, window: int = 0, sinks: int = 0):
    """softmax over what a query sees of (q k^T / sqrt(D)), times v: query i sees key j <= i where i - j < ``window`` or j <
    ``sinks`` (``window`` 0: all).  ``qkv`` [batch * seq, kv_heads * (group + 2) * D], any ``seq``.  Returns
    (out [batch * seq, kv_heads * group * D], lse [batch, kv_heads * group, seq])."""
    D = _check(qkv, batch, seq, kv_heads, group, window, sinks)
    heads = kv_heads * group
    window, sinks = min(window, seq), min(sinks, seq)          # (more is the whole sequence, and might not fit the kernels' 32 bits)
    if qkv.is_cuda:
        stream, device = _native.stream_on(qkv.get_device()), qkv.device
        out = torch.empty(batch * seq, heads * D, dtype=qkv.dtype, device=device)
        lse = torch.empty(batch, heads, seq, dtype=torch.float32, device=device)
        if batch:
            x = _dense(qkv)
            _native.load().window_attention_fwd(x.data_ptr(), out.data_ptr(), lse.data_ptr(), batch, seq, kv_heads, group, window, sinks,
                                                _SCALE, _native.status().dev, stream)
        return out, lse
    q, k, v, s = _formulation(qkv, batch, seq, kv_heads, group, window, sinks, D)
    o = torch.softmax(s, -1) @ v
    return o.permute(0, 3, 1, 2, 4).reshape(batch * seq, heads * D).to(qkv.dtype), torch.logsumexp(s, -1).view(batch, heads, seq)


def window_attention_bwd(dout, qkv, out, lse, batch: int, seq: int, kv_heads: int, group: int = 1, window: int = 0, sinks: int = 0):
    """Gradient of ``qkv`` in its layout; shared key/value heads get the sum over their query heads."""
    D = _check(qkv, batch, seq, kv_heads, group, window, sinks)
    heads = kv_heads * group
    window, sinks = min(window, seq), min(sinks, seq)
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != (batch * seq, heads * D) or t.dtype is not qkv.dtype or t.get_device() != qkv.get_device():
            raise ValueError(f"{name} must be {qkv.dtype} [{batch * seq}, {heads * D}] beside qkv (got {t.dtype} {tuple(t.shape)} on {t.device})")
    if lse.shape != (batch, heads, seq) or lse.dtype is not torch.float32 or lse.get_device() != qkv.get_device():
        raise ValueError(f"lse must be fp32 [{batch}, {heads}, {seq}] beside qkv (got {lse.dtype} {tuple(lse.shape)} on {lse.device})")
    if qkv.is_cuda:
        stream = _native.stream_on(qkv.get_device())
        dqkv = torch.empty_like(qkv) if qkv.is_contiguous() else torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        if batch:
            scratch = torch.empty(_scratch(batch, seq, kv_heads, group, window, sinks), dtype=torch.float32, device=qkv.device)
            x, o, do, l = _dense(qkv), _dense(out), _dense(dout), _dense(lse)
            _native.load().window_attention_bwd(x.data_ptr(), o.data_ptr(), do.data_ptr(), l.data_ptr(), dqkv.data_ptr(), scratch.data_ptr(),
                                                batch, seq, kv_heads, group, window, sinks, _SCALE, _native.status().dev, stream)
        return dqkv
    q, k, v, s = _formulation(qkv, batch, seq, kv_heads, group, window, sinks, D)
    rows_of = lambda t: t.float().view(batch, seq, kv_heads, group, D).permute(0, 2, 3, 1, 4)
    do, o, scale = rows_of(dout), rows_of(out), 1.0 / math.sqrt(D)
    p = torch.exp(s - lse.view(batch, kv_heads, group, seq, 1))
    dv = (p.transpose(-1, -2) @ do).sum(2, keepdim=True)
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    return torch.cat([ds @ k, dk, dv], 2).permute(0, 3, 1, 2, 4).reshape(qkv.shape).to(qkv.dtype)


# ----------------------------------------------------------------------------------------------
# single tokens over a cache of fixed size
# ----------------------------------------------------------------------------------------------
class WindowCache:
    """Keys and values [batch, kv_heads, sinks + window, head_dim] of what the next token of each sequence sees: position p lies in
    slot p below ``sinks`` and in slot sinks + (p - sinks) % window from there on.  Whatever a slot holds before its first position
    is stored is never used."""

    def __init__(self, k, v, window: int, sinks: int = 0):
        if window < 1 or sinks < 0:
            raise ValueError(f"a cache needs window >= 1 and sinks >= 0 (got {window}, {sinks})")
        if (k.dim() != 4 or k.shape[1] < 1 or k.shape[2] != window + sinks or k.shape[3] < 1 or v.shape != k.shape or v.dtype != k.dtype
                or v.device != k.device):
            raise ValueError(f"keys and values must both be [batch, kv_heads >= 1, {window + sinks}, head_dim >= 1] (got {tuple(k.shape)} {k.dtype} "
                             f"and {tuple(v.shape)} {v.dtype})")
        if k.is_cuda:
            if k.dtype != torch.bfloat16 or k.shape[3] != HEAD_DIM:
                raise ValueError(f"the kernel needs a bf16 cache with head_dim {HEAD_DIM} (got {k.dtype}, {k.shape[3]})")
            if not (k.is_contiguous() and v.is_contiguous()) or k.data_ptr() % 16 or v.data_ptr() % 16:
                raise ValueError("the kernel needs contiguous caches on 16-byte boundaries")
        self._k, self._v, self.window, self.sinks = k, v, window, sinks
        self._work = {}
        self._scale = 1.0 / math.sqrt(k.shape[3])

    # (the tensors stay those that were checked)
    @property
    def k(self):
        return self._k

    @property
    def v(self):
        return self._v

    @classmethod
    def new(cls, batch: int, kv_heads: int, window: int, sinks: int = 0, head_dim: int = HEAD_DIM, dtype=torch.bfloat16, device=None):
        k, v = (torch.zeros(batch, kv_heads, sinks + window, head_dim, dtype=dtype, device=device) for _ in range(2))
        return cls(k, v, window, sinks)

    def slots(self, positions):
        return torch.where(positions < self.sinks, positions, self.sinks + (positions - self.sinks) % self.window)

    def fill(self, qkv, seq: int, group: int = 1):
        """Keys and values of the first ``seq`` tokens of every sequence, as far as later tokens see them; ``qkv`` [batch * seq, ...]."""
        batch, kv = self.k.shape[:2]
        D = _width(qkv, kv, group, batch * seq)
        if D != self.k.shape[3]:
            raise ValueError(f"the cache holds {self.k.shape[3]} features per head, the rows {D}")
        pos = torch.arange(seq, device=qkv.device)
        pos = torch.cat([pos[: self.sinks], pos[max(self.sinks, seq - self.window):]])
        x = qkv.reshape(batch, seq, kv, group + 2, D)[:, pos]
        at = self.slots(pos)
        self.k[:, :, at] = x[:, :, :, group].transpose(1, 2)
        self.v[:, :, at] = x[:, :, :, group + 1].transpose(1, 2)

    def workspace(self, group: int):
        """(splits, partial results, counters) of the decoding kernel, laid out once (by a graph that is being captured, where nothing
        is laid out yet, for itself: its counters are zeroed when it runs, not now)."""
        work = self._work.get(group)
        if work is None:
            batch, kv, slots = self.k.shape[:3]
            C = _native.load()
            sms = torch.cuda.get_device_properties(self.k.device).multi_processor_count
            splits = C.window_decode_splits(batch, kv, group, slots, sms)
            units = batch * kv * -(-group // 16) if splits > C.WINDOW_DECODE_CLUSTER else 0      # (fewer are joined without)
            parts = torch.empty(units * splits * C.WINDOW_DECODE_PART, dtype=torch.float32, device=self.k.device)
            counters = torch.zeros(units, dtype=torch.int32, device=self.k.device)
            work = (splits, parts, counters)
            if units == 0 or not torch.cuda.is_current_stream_capturing():
                self._work[group] = work
        return work


def _decode(x, pitch: int, cache: WindowCache, positions, batch: int, kv: int, group: int, D: int):
    stream = _native.stream_on(x.get_device())
    out = torch.empty(batch, kv * group * D, dtype=x.dtype, device=x.device)
    splits, parts, counters = cache.workspace(group)
    _native.load().window_decode(x.data_ptr(), pitch, cache.k.data_ptr(), cache.v.data_ptr(), positions.data_ptr(), out.data_ptr(), batch,
                                 kv, group, cache.window, cache.sinks, cache._scale, parts.data_ptr(), counters.data_ptr(), splits,
                                 stream)
    return out


def window_attention_decode(qkv, cache: WindowCache, positions, group: int = 1):
    """Attention of one token per sequence, ``qkv`` [batch, kv_heads * (group + 2) * D], at ``positions`` (int64 [batch]) over what
    it sees, itself included.  Stores its key and value in the cache.  A negative position is an idle sequence: nothing is
    stored, its output is zero.  Returns [batch, kv_heads * group * D]."""
    k = cache.k
    batch, kv, slots, D = k.shape
    # the common call, checked in a few steps: a kernel of a few us is over before a longer list of them
    if (k.is_cuda and group > 0 and qkv.shape == (batch, kv * (group + 2) * D) and qkv.dtype is k.dtype and qkv.is_contiguous()
            and qkv.data_ptr() & 15 == 0 and positions.dtype is torch.int64 and positions.shape == (batch,) and positions.is_contiguous()
            and qkv.get_device() == positions.get_device() == k.get_device() and batch):
        return _decode(qkv, qkv.shape[1], cache, positions, batch, kv, group, D)
    if _width(qkv, kv, group, batch) != D:
        raise ValueError(f"the cache holds {D} features per head, the rows {qkv.shape[1] // (kv * (group + 2))}")
    if positions.shape != (batch,) or positions.dtype != torch.int64 or positions.device != qkv.device:
        raise ValueError(f"positions must be int64 [{batch}] beside the rows (got {positions.dtype} {tuple(positions.shape)} on "
                         f"{positions.device})")
    if qkv.dtype != cache.k.dtype or qkv.device != cache.k.device:
        raise ValueError(f"rows are {qkv.dtype} on {qkv.device}, the cache {cache.k.dtype} on {cache.k.device}")
    if qkv.is_cuda:
        if batch == 0:
            return qkv.new_empty(0, kv * group * D)
        x = rows.as_aligned(qkv)
        return _decode(x, rows.pitch(x), cache, positions.contiguous(), batch, kv, group, D)
    x = qkv.view(batch, kv, group + 2, D)
    out = torch.zeros(batch, kv, group, D, dtype=torch.float32)
    for b, p in enumerate(positions.tolist()):
        if p < 0:
            continue
        s = p if p < cache.sinks else cache.sinks + (p - cache.sinks) % cache.window
        cache.k[b, :, s], cache.v[b, :, s] = x[b, :, group], x[b, :, group + 1]
        held = min(p + 1, slots)
        w = torch.softmax(x[b, :, :group].float() @ cache.k[b, :, :held].float().transpose(-1, -2) / math.sqrt(D), -1)
        out[b] = w @ cache.v[b, :, :held].float()
    return out.view(batch, -1).to(qkv.dtype)
