"""Token by token through a windowed GPT on one device: every block keeps what the next token sees in a cache of fixed size."""
from __future__ import annotations

import torch

from ..ops import functional as F
from ..ops.window import WindowCache
from ..parallel.mesh import ShardedTensor
from .gpt import GPTModel


class GPTDecoder:
    """``prefill`` takes prompts of one length, ``step`` a token of each sequence at its own position; both return logits
    [batch, vocab] of the next tokens.  A negative position is an idle sequence, whose token and logits mean nothing.

    Tokens and positions are int64 on the model's device.  What they hold is checked on the CPU; on a GPU, where that would wait for the
    device, a token outside the vocabulary counts as the nearest one in it, and a position that a model with learned positions has
    no vector for (``cfg.seq`` and beyond) makes the logits of its sequence NaN."""

    def __init__(self, model: GPTModel, batch: int):
        cfg, mesh = model.cfg, model.mesh
        if mesh.R * mesh.C != 1:
            raise ValueError("decoding runs on one device (a 1 x 1 mesh)")
        if cfg.window < 1:
            raise ValueError("decoding needs a model with a window: its cache has a fixed size")
        if "rs" in cfg.dataflows:
            raise ValueError("decoding takes the layers' inputs as [tokens, features]: no 'rs' dataflow")
        self.model, self.cfg, self.batch, self.key = model, cfg, batch, next(iter(mesh.coords()))
        self.kv = cfg.kv_heads or cfg.n_heads
        self.group = cfg.n_heads // self.kv
        self.caches = [WindowCache.new(batch, self.kv, cfg.window, cfg.sinks, cfg.d_model // cfg.n_heads, cfg.dtype, model.device)
                       for _ in model.blocks]

    def _linear(self, layer, x):
        return layer.forward(ShardedTensor(self.model.mesh, {self.key: x}), keep=False).shards[self.key]

    def _norm(self, layer, x, res):
        return F.ln_full(x, res, layer.gamma.shards[self.key], layer.bias.shards[self.key], layer.eps)[:2]

    def _run(self, x, attend):
        """Rows of activations through the blocks; ``attend(i, qkv)`` is block i's attention."""
        delta = None
        for i, b in enumerate(self.model.blocks):
            h, y = self._norm(b.ln1, x, delta)
            a = self._linear(b.out_proj, attend(i, self._linear(b.in_proj, y)))
            x, y = self._norm(b.ln2, a, h)
            if b.ff is not None:
                delta = self._linear(b.ff, y)
            else:
                delta = self._linear(b.ff2, F.gelu(self._linear(b.ff1, y)))
        return x, delta

    def _logits(self, x, delta):
        return self._linear(self.model.head, self._norm(self.model.ln_f, x, delta)[1])[:, :self.cfg.vocab]

    def _check(self, name, t, shape):
        device = self.model.tok.shards[self.key].device
        if t.shape != shape or t.dtype != torch.int64 or t.device != device:
            raise ValueError(f"{name} must be int64 {list(shape)} on {device} (got {t.dtype} {list(t.shape)} on {t.device})")

    def _embed(self, tokens, positions):
        tok = self.model.tok.shards[self.key]
        rows = tok.shape[0]
        if not tok.is_cuda and ((tokens < 0) | (tokens >= rows))[positions >= 0].any():
            raise ValueError(f"tokens must be in [0, {rows})")
        tokens = tokens.clamp(0, rows - 1).contiguous()
        if self.model.pos is None:
            return F.embedding_fwd(tokens, tok, None, 1)
        pos = self.model.pos.shards[self.key]
        beyond = positions >= pos.shape[0]
        if not tok.is_cuda and beyond.any():
            raise ValueError(f"the model has learned positions below {pos.shape[0]} (got {int(positions.max())})")
        x = (tok[tokens].float() + pos[positions.clamp(0, pos.shape[0] - 1)].float()).to(tok.dtype)
        return x.masked_fill_(beyond[:, None], float("nan"))

    def prefill(self, tokens):
        """``tokens`` [batch, n], positions 0 .. n - 1."""
        if tokens.dim() != 2 or tokens.shape[0] != self.batch or tokens.shape[1] < 1:
            raise ValueError(f"prompts must be [{self.batch}, n >= 1] (got {tuple(tokens.shape)})")
        n, cfg = tokens.shape[1], self.cfg
        self._check("prompts", tokens, (self.batch, n))
        if self.model.pos is not None and n > cfg.seq:
            raise ValueError(f"the model has learned positions of {cfg.seq} tokens (got a prompt of {n})")
        pos = torch.arange(n, device=tokens.device).repeat(self.batch)

        def attend(i, qkv):
            rot = self.model.blocks[i].attn.rotary
            if rot is not None:
                F.rotary_qkv(qkv, rot, self.kv, self.group, seq=n, out=qkv)
            self.caches[i].fill(qkv, n, self.group)
            return F.window_attention_fwd(qkv, self.batch, n, self.kv, self.group, cfg.window, cfg.sinks)[0]

        x, delta = self._run(self._embed(tokens.reshape(-1), pos), attend)
        last = lambda t: t.view(self.batch, n, -1)[:, -1].contiguous()
        return self._logits(last(x), last(delta))

    def step(self, tokens, positions):
        """``tokens``, ``positions`` int64 [batch]."""
        self._check("tokens", tokens, (self.batch,))
        self._check("positions", positions, (self.batch,))

        def attend(i, qkv):
            rot = self.model.blocks[i].attn.rotary
            if rot is not None:
                F.rotary_qkv(qkv, rot, self.kv, self.group, positions=positions, out=qkv)
            return F.window_attention_decode(qkv, self.caches[i], positions, self.group)

        return self._logits(*self._run(self._embed(tokens, positions), attend))
