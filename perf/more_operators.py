"""The operators of a decoder's training step as timed cases: the gated feed-forward block, the loss of its output head without the
logits in memory, and the orthogonal update of its matrices.

``listed()`` are the standing cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` builds what a program
holds before the call, ``run`` is one pass, ``work`` the bytes and operations it cannot do without, ``exact`` the same
outputs in 64 bits.  With ``own`` set, ``run`` calls the framework's operators; otherwise it computes them by elementary
operations in 32 bits, rounded once at the end.

16-bit data is bf16.  A weight of layout 'nn' lies as [inputs, outputs], one of 'nt' as [outputs, inputs].
"""
from __future__ import annotations

import math
import random

import torch

own = False

VOCAB_PAD = 2048                          # columns of a head that lies as [inputs, outputs] are a multiple of this
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # of x, x^3 and x^5
MOST = 1.05e13                            # operations of the largest case


# ----------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------
def listed():
    return [
        # the next token of eight sequences of a model that answers: latency, and the weights have to be read
        {"name": "gated_tokens", "kind": "gated", "tokens": 8, "width": 1024, "ffn": 2816, "act": "silu", "down": "nt", "train": False},
        # a training step of a small model on one short batch
        {"name": "gated_small", "kind": "gated", "tokens": 200, "width": 512, "ffn": 1408, "act": "silu", "down": "nn", "train": True},
        # a micro-batch of 4 x 2048 tokens of the 6.7B-parameter decoder, with the parameters of its feed-forward block
        {"name": "gated_train", "kind": "gated", "tokens": 8192, "width": 4096, "ffn": 10752, "act": "silu", "down": "nt", "train": True},
        # nothing is a multiple of a tile; the other activation
        {"name": "gated_ragged", "kind": "gated", "tokens": 1999, "width": 1032, "ffn": 2744, "act": "gelu", "down": "nn", "train": True},
        # the loss of a small model on one short batch
        {"name": "head_small", "kind": "head", "rows": 128, "width": 512, "vocab": 1000, "layout": "nn", "missing": False, "train": True},
        # the loss of a micro-batch of 4 x 2048 tokens of the 6.7B-parameter decoder
        {"name": "head_train", "kind": "head", "rows": 8192, "width": 4096, "vocab": 50257, "layout": "nn", "missing": False,
         "train": True},
        # a head that lies as an embedding table does; odd sizes, tokens without a label
        {"name": "head_ragged", "kind": "head", "rows": 2047, "width": 1032, "vocab": 30011, "layout": "nt", "missing": True,
         "train": True},
        # scoring text: the losses alone
        {"name": "head_score", "kind": "head", "rows": 4096, "width": 1024, "vocab": 50257, "layout": "nn", "missing": False,
         "train": False},
        # one small matrix: latency
        {"name": "orthogonal_small", "kind": "orthogonal", "batch": 1, "rows": 256, "cols": 256, "type": "float32"},
        # the same projection of eight layers at once
        {"name": "orthogonal_layers", "kind": "orthogonal", "batch": 8, "rows": 1024, "cols": 1024, "type": "float32"},
        # taller than wide, no multiple of a tile, gradients in 16 bits
        {"name": "orthogonal_tall", "kind": "orthogonal", "batch": 3, "rows": 1000, "cols": 520, "type": "bfloat16"},
        # the first feed-forward matrix of the 6.7B-parameter decoder
        {"name": "orthogonal_large", "kind": "orthogonal", "batch": 1, "rows": 4096, "cols": 16384, "type": "float32"},
    ]


def _log(rng: random.Random, lo: int, hi: int, step: int = 1) -> int:
    """A multiple of ``step`` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng: random.Random):
    kind = rng.choice(["gated", "head", "orthogonal"])
    if kind == "gated":
        train = rng.random() < 0.7
        case = {"kind": kind, "tokens": _log(rng, 1, 16384), "width": _log(rng, 64, 4096, 8), "ffn": _log(rng, 64, 10752, 8),
                "act": rng.choice(["silu", "gelu"]), "down": rng.choice(["nn", "nt"]), "train": train}
    elif kind == "head":
        case = {"kind": kind, "rows": _log(rng, 1, 16384), "width": _log(rng, 64, 4096, 8), "vocab": _log(rng, 200, 128000),
                "layout": rng.choice(["nn", "nt"]), "missing": rng.random() < 0.4, "train": rng.random() < 0.7}
    else:
        case = {"kind": kind, "batch": _log(rng, 1, 16), "rows": _log(rng, 8, 4096), "cols": _log(rng, 8, 16384),
                "type": rng.choice(["float32", "float32", "bfloat16"])}
        if rng.random() < 0.3:
            case["rows"], case["cols"] = case["cols"], case["rows"]
        most = max(1, int(1.6e8 // (case["rows"] * case["cols"])))
        case["batch"] = min(case["batch"], most)
    first = {"gated": "tokens", "head": "rows", "orthogonal": "batch"}[kind]
    over = _cost(case) / MOST
    if over > 1:
        case[first] = max(1, int(case[first] / over))
    return case


# ----------------------------------------------------------------------------------------------
# inputs, made from the seed alone
# ----------------------------------------------------------------------------------------------
class _Source:
    def __init__(self, seed: int):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=self.g)

    def ids(self, low, high, *shape):
        return torch.randint(low, high, shape, device="cuda", generator=self.g)


def _columns(case):
    """Output features of a head: the vocabulary, padded where the head lies as [inputs, outputs]."""
    return -(-case["vocab"] // VOCAB_PAD) * VOCAB_PAD if case["layout"] == "nn" else case["vocab"]


def _inputs(case, seed):
    src, k = _Source(seed), case["kind"]
    if k == "gated":
        n, d, f = case["tokens"], case["width"], case["ffn"]
        s = {"x": src.normal(n, d), "gate": src.normal(d, f, std=d ** -0.5), "up": src.normal(d, f, std=d ** -0.5),
             "down": src.normal(*((f, d) if case["down"] == "nn" else (d, f)), std=f ** -0.5)}
        if case["train"]:
            s["dy"] = src.normal(n, d, std=0.01)
        return s
    if k == "head":
        n, d, cols = case["rows"], case["width"], _columns(case)
        w = src.normal(*((d, cols) if case["layout"] == "nn" else (cols, d)), std=2 * d ** -0.5)
        targets = src.ids(0, case["vocab"], n)
        x = src.normal(n, d)
        # half of the tokens are predicted with some confidence
        told = (w[:, targets].T if case["layout"] == "nn" else w[targets]).float() * 1.5
        x = (x.float() + told * (torch.arange(n, device="cuda") % 2)[:, None]).to(torch.bfloat16)
        if case["missing"]:
            targets[3::11] = -1
        return {"x": x, "w": w, "targets": targets}
    # gradients of a layer: some directions carry most of the norm
    b, m, n = case["batch"], case["rows"], case["cols"]
    r = max(1, min(m, n) // 16)
    g = src.normal(b, m, r, dtype=torch.float32) @ src.normal(b, r, n, std=r ** -0.5, dtype=torch.float32)
    g += src.normal(b, m, n, std=0.3, dtype=torch.float32)
    return {"g": g.mul_(1e-4).to(getattr(torch, case["type"]))}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    return s


# ----------------------------------------------------------------------------------------------
# a pass
# ----------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"gated": _plain_gated, "head": _plain_head, "orthogonal": _plain_orthogonal}[kind](s)
    from meshslice_b200.ops import functional as F
    if kind == "gated":
        w = (s["gate"], s["up"], s["down"])
        y, saved = F.gated_ff_fwd(s["x"], *w, act=case["act"], down_layout=case["down"], keep=case["train"])
        if not case["train"]:
            return {"y": y}
        dx, (dgate, dup, ddown) = F.gated_ff_bwd(s["dy"], s["x"], *w, saved, act=case["act"], down_layout=case["down"])
        return {"y": y, "dx": dx, "dgate": dgate, "dup": dup, "ddown": ddown}
    if kind == "head":
        if not case["train"]:
            return {"loss": F.head_loss(s["x"], s["w"], s["targets"], case["vocab"], layout=case["layout"])}
        loss, dx, dw = F.head_loss_grad(s["x"], s["w"], s["targets"], case["vocab"], 1.0 / case["rows"], layout=case["layout"])
        return {"loss": loss, "dx": dx, "dw": dw}
    return F.orthogonalize(s["g"], steps=5, coefficients=COEFFICIENTS)


# ----------------------------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits
# ----------------------------------------------------------------------------------------------
def _plain_gated(s):
    case = s["case"]
    x, wg, wu, wd = s["x"].float(), s["gate"].float(), s["up"].float(), s["down"].float()
    if case["down"] == "nt":
        wd = wd.T
    g, u = x @ wg, x @ wu
    if case["act"] == "silu":
        e = 1 / (1 + (-g).exp())
        a = g * e
        da = e * (1 + g * (1 - e))
    else:
        c = math.sqrt(2 / math.pi)
        e = (c * (g + 0.044715 * g * g * g)).tanh()
        a = 0.5 * g * (1 + e)
        da = 0.5 * (1 + e) + 0.5 * g * (1 - e * e) * c * (1 + 3 * 0.044715 * g * g)
    h = a * u
    out = {"y": h @ wd}
    if case["train"]:
        dy = s["dy"].float()
        dh = dy @ wd.T
        dg, du = dh * u * da, dh * a
        ddown = h.T @ dy
        out |= {"dx": dg @ wg.T + du @ wu.T, "dgate": x.T @ dg, "dup": x.T @ du, "ddown": ddown if case["down"] == "nn" else ddown.T}
    return {k: v.to(s["x"].dtype).contiguous() for k, v in out.items()}


def _plain_head(s):
    case = s["case"]
    vocab, n = case["vocab"], case["rows"]
    x, w = s["x"].float(), (s["w"] if case["layout"] == "nn" else s["w"].T)[:, :vocab].float()
    label = (s["targets"] >= 0) & (s["targets"] < vocab)
    y = torch.where(label, s["targets"], 0)[:, None]
    z = x @ w
    z -= z.amax(1, keepdim=True)
    zy = z.gather(1, y)
    p = z.exp_()
    total = p.sum(1, keepdim=True)
    loss = torch.where(label, (total.log() - zy)[:, 0], 0.0)
    if not case["train"]:
        return {"loss": loss}
    p *= label[:, None] / (n * total)
    p.scatter_add_(1, y, -label[:, None].float() / n)
    dw = torch.zeros(case["width"], _columns(case), device="cuda")
    dw[:, :vocab] = x.T @ p
    dx = p @ w.T
    return {"loss": loss, "dx": dx.to(s["x"].dtype), "dw": (dw if case["layout"] == "nn" else dw.T).to(s["w"].dtype).contiguous()}


def _plain_orthogonal(s):
    g = s["g"].float()
    tall = g.shape[1] > g.shape[2]
    x = g.transpose(1, 2) if tall else g
    x = x / x.square().sum((1, 2), keepdim=True).sqrt()
    a, b, c = COEFFICIENTS
    for _ in range(5):
        q = x @ x.transpose(1, 2)
        x = a * x + (b * q + c * (q @ q)) @ x
    return (x.transpose(1, 2) if tall else x).to(torch.bfloat16).contiguous()


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------
def work(case):
    k = case["kind"]
    if k == "gated":
        n, d, f = case["tokens"], case["width"], case["ffn"]
        if case["train"]:
            return {"bytes": 2 * (4 * n * d + 6 * d * f), "flops": 18 * n * d * f}
        return {"bytes": 2 * (2 * n * d + 3 * d * f), "flops": 6 * n * d * f}
    if k == "head":
        n, d, v = case["rows"], case["width"], case["vocab"]
        if case["train"]:
            return {"bytes": 2 * (2 * n * d + d * v + d * _columns(case)) + 12 * n, "flops": 6 * n * d * v}
        return {"bytes": 2 * (n * d + d * v) + 12 * n, "flops": 2 * n * d * v}
    b, m, n = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # of a symmetric product one half has to be computed
    return {"bytes": b * m * n * (6 if case["type"] == "float32" else 4), "flops": 5 * b * (3 * m * m * n + m * m * m)}


def _cost(case):
    """Operations, or those for which the card would have time while it moves the bytes."""
    w = work(case)
    return max(w["flops"], 250 * w["bytes"])


# ----------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    return {"gated": _exact_gated, "head": _exact_head, "orthogonal": _exact_orthogonal}[case["kind"]](case, s)


def _exact_gated(case, s):
    """The gradients by automatic differentiation of the block's formula."""
    leaf = {k: s[k].double().requires_grad_(case["train"]) for k in ("x", "gate", "up", "down")}
    g = leaf["x"] @ leaf["gate"]
    if case["act"] == "silu":
        a = g * torch.sigmoid(g)
    else:
        a = g / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * g * (1 + 0.044715 * g ** 2)))
    h = a * (leaf["x"] @ leaf["up"])
    y = torch.einsum("nf,fd->nd" if case["down"] == "nn" else "nf,df->nd", h, leaf["down"])
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [leaf[k] for k in ("x", "gate", "up", "down")], s["dy"].double())
    return {"y": y.detach(), "dx": grads[0], "dgate": grads[1], "dup": grads[2], "ddown": grads[3]}


def _exact_head(case, s):
    """Piece by piece of the rows: log-softmax, the dense difference to the labels, the gradients of the two factors."""
    n, vocab = case["rows"], case["vocab"]
    w = s["w"].double()
    if case["layout"] == "nt":
        w = w.T
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    dx = torch.zeros(n, case["width"], dtype=torch.float64, device="cuda")
    dw = torch.zeros(case["width"], w.shape[1], dtype=torch.float64, device="cuda")
    for i in range(0, n, 2048):
        x, t = s["x"][i:i + 2048].double(), s["targets"][i:i + 2048]
        at = ((t >= 0) & (t < vocab)).nonzero()[:, 0]
        logp = torch.log_softmax(x @ w[:, :vocab], 1)
        loss[i + at] = -logp[at, t[at]]
        if case["train"]:
            d = torch.zeros_like(logp)
            d[at] = logp[at].exp()
            d[at, t[at]] -= 1
            d /= n
            dx[i:i + 2048] = d @ w[:, :vocab].T
            dw[:, :vocab] += x.T @ d
    if not case["train"]:
        return {"loss": loss}
    return {"loss": loss, "dx": dx, "dw": dw if case["layout"] == "nn" else dw.T.contiguous()}


def _exact_orthogonal(case, s):
    """Matrix by matrix: an odd polynomial of the singular values, by Horner's rule on the smaller Gram matrix."""
    a, b, c = COEFFICIENTS
    out = torch.empty(case["batch"], case["rows"], case["cols"], dtype=torch.float64, device="cuda")
    one = torch.eye(min(case["rows"], case["cols"]), dtype=torch.float64, device="cuda")
    for i in range(case["batch"]):
        x = s["g"][i].double()
        x = x / torch.linalg.norm(x)
        for _ in range(5):
            if case["rows"] <= case["cols"]:
                q = x @ x.T
                x = (a * one + q @ (b * one + c * q)) @ x
            else:
                q = x.T @ x
                x = x @ (a * one + q @ (b * one + c * q))
        out[i] = x
    return out
