"""The operators of a long-context decoder as timed cases: rotary positions, attention within a window that keeps the first
tokens visible (training and single tokens over a cache of fixed size), and the loss that trains it from a teacher's top logits.

``listed()`` are the standing cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` builds what a program
holds before the call, ``run`` is one pass, ``work`` the bytes and operations it cannot do without, ``exact`` the same
outputs in 64 bits.  With ``own`` set, ``run`` calls the framework's operators; otherwise it computes them by elementary
operations in 32 bits, rounded once at the end.

Sizes: ``kv`` key/value heads of 128 features, ``group`` query heads that share one; rows of activations hold, per key/value
head, [q_0 | .. | q_group-1 | k | v].  16-bit data is bf16.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128
VOCAB_PAD = 2048
MOST = 4.8e11     # operations of the largest attention case


# ----------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------
def listed():
    return [
        # positions of the tokens that eight sequences are at, far into a context scaled to 16 times its trained length: latency
        {"name": "rotary_tokens", "kind": "rotary", "batch": 8, "seq": 1, "kv": 8, "group": 4, "rot": 128, "layout": "half",
         "scaling": "by_parts", "factor": 16.0, "far": 131072, "inverse": False},
        # the projection of a micro-batch of 4 x 2048 tokens of the 6.7B-parameter decoder
        {"name": "rotary_train", "kind": "rotary", "batch": 4, "seq": 2048, "kv": 32, "group": 1, "rot": 128, "layout": "half",
         "scaling": "none", "factor": 1.0, "far": 0, "inverse": False},
        # its gradient, in the other layout, for half of the head, odd lengths and shared heads
        {"name": "rotary_grad_ragged", "kind": "rotary", "batch": 3, "seq": 1999, "kv": 6, "group": 3, "rot": 64,
         "layout": "interleaved", "scaling": "linear", "factor": 4.0, "far": 0, "inverse": True},
        # a training step of a small model on one short sequence that fills no tile
        {"name": "window_short", "kind": "window", "batch": 1, "seq": 200, "kv": 2, "group": 1, "window": 64, "sinks": 0,
         "train": True},
        # a training step of the decoder above with a window of a quarter of the sequence
        {"name": "window_train", "kind": "window", "batch": 4, "seq": 2048, "kv": 32, "group": 1, "window": 512, "sinks": 4,
         "train": True},
        # training on longer sequences with shared key/value heads; nothing is a multiple of a tile
        {"name": "window_train_grouped", "kind": "window", "batch": 2, "seq": 5003, "kv": 4, "group": 4, "window": 1000,
         "sinks": 16, "train": True},
        # scoring a long document: forward only
        {"name": "window_long", "kind": "window", "batch": 1, "seq": 16384, "kv": 4, "group": 4, "window": 4096, "sinks": 4,
         "train": False},
        # a token of one sequence: latency
        {"name": "decode_one", "kind": "decode", "batch": 1, "kv": 8, "group": 4, "window": 1024, "sinks": 4, "low": 700,
         "high": 700},
        # a token of each of 64 sequences, from the first one to far beyond the window
        {"name": "decode_many", "kind": "decode", "batch": 64, "kv": 8, "group": 4, "window": 4096, "sinks": 4, "low": 0,
         "high": 20000},
        # the loss of a small model on one short batch
        {"name": "distill_small", "kind": "distill", "rows": 128, "vocab": 1000, "top": 8, "temperature": 1.0, "hard": 0.0,
         "missing": False},
        # the loss of a micro-batch over a 50k vocabulary, softened, half of it from the labels
        {"name": "distill_train", "kind": "distill", "rows": 4096, "vocab": 50257, "top": 64, "temperature": 2.0, "hard": 0.5,
         "missing": False},
        # odd sizes, teachers that kept fewer logits than others, positions without any
        {"name": "distill_ragged", "kind": "distill", "rows": 2047, "vocab": 30011, "top": 33, "temperature": 1.0, "hard": 0.1,
         "missing": True},
    ]


def _log(rng: random.Random, lo: int, hi: int, step: int = 1) -> int:
    """A multiple of ``step`` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng: random.Random):
    kind = rng.choice(["rotary", "window", "window", "decode", "distill"])
    if kind == "rotary":
        kv, group = _log(rng, 1, 32), rng.choice([1, 1, 2, 3, 4, 8])
        kv = max(1, min(kv, 96 // (group + 2)))
        seq = _log(rng, 1, 4096)
        most = max(1, 4 * 2048 * 96 // (seq * kv * (group + 2)))
        return {"kind": kind, "batch": _log(rng, 1, min(64, most)), "seq": seq, "kv": kv, "group": group,
                "rot": rng.choice([32, 64, 96, 128, 128]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "base", "by_parts"]), "factor": rng.choice([2.0, 4.0, 16.0]),
                "far": rng.choice([0, 0, 131072]), "inverse": rng.random() < 0.5}
    if kind == "window":
        seq = _log(rng, 1, 16384)
        kv, group = _log(rng, 1, 16), rng.choice([1, 1, 2, 3, 4, 8])
        window = _log(rng, 1, 4096) if rng.random() < 0.8 else 0
        case = {"kind": kind, "batch": 1, "seq": seq, "kv": 1, "group": group, "window": window,
                "sinks": rng.choice([0, 1, 4, 4, 16, 130]), "train": rng.random() < 0.7}
        if _cost(case) > MOST:
            case["group"] = group = 1
        most = max(1, int(MOST // _cost(case)))                    # heads and sequences that the largest listed case's work is
        case["kv"] = kv = max(1, min(kv, most, 96 // group))
        case["batch"] = _log(rng, 1, max(1, min(8, most // kv, 65536 // seq)))
        return case
    if kind == "decode":
        kv, group, window = _log(rng, 1, 16), rng.choice([1, 2, 3, 4, 7, 8, 16]), _log(rng, 1, 8192)
        high = _log(rng, 1, 4 * window)
        most = max(1, 64 * 8 * 4096 // (kv * max(window, 64)))
        return {"kind": kind, "batch": _log(rng, 1, min(most, 256)), "kv": kv, "group": group, "window": window,
                "sinks": rng.choice([0, 1, 4, 16]), "low": rng.randint(0, high), "high": high}
    rows, vocab = _log(rng, 1, 4096), _log(rng, 200, 50257)
    return {"kind": kind, "rows": rows, "vocab": vocab, "top": _log(rng, 1, 128), "temperature": rng.choice([1.0, 1.0, 2.0, 0.7, 4.0]),
            "hard": rng.choice([0.0, 0.1, 0.5, 1.0]), "missing": rng.random() < 0.4}


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

    def order(self, n):
        return torch.randperm(n, device="cuda", generator=self.g)


def _width(case):
    return case["kv"] * (case["group"] + 2) * D


def _stops(case):
    """Positions of the sequences of a decoding step, evenly from the lowest to the highest."""
    n, lo, hi = case["batch"], case["low"], case["high"]
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _inputs(case, seed):
    src, k = _Source(seed), case["kind"]
    if k == "rotary":
        s = {"x": src.normal(case["batch"] * case["seq"], _width(case))}
        if case["far"]:
            first = src.ids(0, case["far"], case["batch"])
            s["positions"] = (first[:, None] + torch.arange(case["seq"], device="cuda")).reshape(-1)
        return s
    if k == "window":
        t = case["batch"] * case["seq"]
        s = {"qkv": src.normal(t, _width(case))}
        if case["train"]:
            s["dout"] = src.normal(t, case["kv"] * case["group"] * D, std=0.01)
        return s
    if k == "decode":
        slots = case["sinks"] + case["window"]
        stops = torch.tensor(_stops(case), device="cuda")
        return {"qkv": src.normal(case["batch"], _width(case)), "k": src.normal(case["batch"], case["kv"], slots, D),
                "v": src.normal(case["batch"], case["kv"], slots, D), "positions": stops[src.order(case["batch"])]}
    rows, vocab = case["rows"], case["vocab"]
    padded = -(-vocab // VOCAB_PAD) * VOCAB_PAD
    logits = src.normal(rows, padded, std=2.0)
    # a teacher that agrees with the student in part
    values, ids = (logits[:, :vocab].float() * 0.7 + src.normal(rows, vocab, std=1.5)).topk(case["top"], dim=1)
    if case["missing"]:
        kept = src.ids(0, case["top"] + 1, rows)
        kept[::7] = 0
        gone = torch.arange(case["top"], device="cuda")[None, :] >= kept[:, None]
        ids = ids.masked_fill(gone, -1)
    targets = src.ids(0, vocab, rows)
    if case["missing"]:
        targets[3::11] = -1
    return {"logits": logits, "ids": ids.contiguous(), "values": values.contiguous(), "targets": targets}


def _settings(case):
    return {"head_dim": D, "rot_dim": case["rot"], "theta": 10000.0, "layout": case["layout"], "scaling": case["scaling"],
            "factor": case["factor"], "original_len": 8192}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "rotary":
        if own:
            from meshslice_b200.ops.rotary import Rotary, RotaryConfig
            s["rotary"] = Rotary(RotaryConfig(**_settings(case)), device="cuda")
        else:
            s["cos"], s["sin"] = _tables(case)
    if case["kind"] == "decode" and own:
        from meshslice_b200.ops.window import WindowCache
        s["cache"] = WindowCache(s["k"], s["v"], window=case["window"], sinks=case["sinks"])
    return s


# ----------------------------------------------------------------------------------------------
# a pass
# ----------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"rotary": _plain_rotary, "window": _plain_window, "decode": _plain_decode, "distill": _plain_distill}[kind](s)
    from meshslice_b200.ops import functional as F
    if kind == "rotary":
        return F.rotary_qkv(s["x"], s["rotary"], case["kv"], case["group"], seq=case["seq"], positions=s.get("positions"),
                            inverse=case["inverse"])
    if kind == "window":
        a = (case["batch"], case["seq"], case["kv"], case["group"], case["window"], case["sinks"])
        out, lse = F.window_attention_fwd(s["qkv"], *a)
        if not case["train"]:
            return {"out": out, "lse": lse}
        return {"out": out, "lse": lse, "dqkv": F.window_attention_bwd(s["dout"], s["qkv"], out, lse, *a)}
    if kind == "decode":
        out = F.window_attention_decode(s["qkv"], s["cache"], s["positions"], case["group"])
        return {"out": out, "k": s["cache"].k, "v": s["cache"].v}
    loss, grad = F.distill_loss_grad(s["logits"], s["ids"], s["values"], case["vocab"], 1.0 / case["rows"],
                                     temperature=case["temperature"], targets=s["targets"], hard_weight=case["hard"])
    return {"loss": loss, "grad": grad}


# ----------------------------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits
# ----------------------------------------------------------------------------------------------
def _tables(case):
    """cos and sin of every position that can come up, times the attention factor of the scaling."""
    c, half = _settings(case), case["rot"] // 2
    theta, s = c["theta"], c["factor"]
    if c["scaling"] == "base":
        theta = theta * s ** (case["rot"] / (case["rot"] - 2))
    f = theta ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    m = 1.0
    if c["scaling"] == "linear":
        f = f / s
    if c["scaling"] == "by_parts":
        turns = c["original_len"] * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        f = f * keep + f / s * (1 - keep)
        m = 0.1 * math.log(s) + 1
    a = torch.arange(case["far"] + case["seq"], dtype=torch.float64, device="cuda")[:, None] * f
    return (a.cos() * m).float(), (a.sin() * m).float()


def _plain_rotary(s):
    case = s["case"]
    tokens, rot, half = case["batch"] * case["seq"], case["rot"], case["rot"] // 2
    pos = s["positions"] if "positions" in s else torch.arange(tokens, device="cuda") % case["seq"]
    cos, sin = s["cos"][pos][:, None, None], s["sin"][pos][:, None, None]
    if case["inverse"]:
        sin = -sin
    x = s["x"].float().view(tokens, case["kv"], case["group"] + 2, D)
    y = x.clone()
    qk = x[:, :, :-1, :rot]
    if case["layout"] == "half":
        a, b = qk[..., :half], qk[..., half:]
        y[:, :, :-1, :half], y[:, :, :-1, half:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = qk[..., 0::2], qk[..., 1::2]
        y[:, :, :-1, 0:rot:2], y[:, :, :-1, 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return y.view(tokens, -1).to(s["x"].dtype)


def _band(t, blocks, size):
    """[b, h, s, D] -> [b, h, blocks, 2 size, D]: each block behind the one before it (zeros before the first); one block alone."""
    b, h, n, d = t.shape
    if blocks == 1:
        return t[:, :, None]
    t = torch.cat([t.new_zeros(b, h, size, d), t, t.new_zeros(b, h, blocks * size - n, d)], 2).view(b, h, blocks + 1, size, d)
    return torch.cat([t[:, :, :-1], t[:, :, 1:]], 3)


def _plain_window(s):
    """Queries in blocks as long as the window, each against its own block of keys, the one before, and the first tokens."""
    case = s["case"]
    b, n, kv, g = case["batch"], case["seq"], case["kv"], case["group"]
    window = min(case["window"] or n, n)
    first, size, scale = min(case["sinks"], n), window, 1.0 / math.sqrt(D)
    blocks, h = -(-n // size), kv * g
    x = s["qkv"].float().view(b, n, kv, g + 2, D)
    rows = lambda t: torch.cat([t, t.new_zeros(b, h, blocks * size - n, D)], 2).view(b, h, blocks, size, D)  # noqa: E731
    q = rows(x[:, :, :, :g].reshape(b, n, h, D).transpose(1, 2))
    k, v = (x[:, :, :, g + i].repeat_interleave(g, 2).transpose(1, 2) for i in (0, 1))
    kw, vw, ks, vs = _band(k, blocks, size), _band(v, blocks, size), k[:, :, None, :first], v[:, :, None, :first]
    qp = torch.arange(blocks * size, device="cuda").view(blocks, size, 1)
    kp = torch.arange(blocks, device="cuda")[:, None, None] * size + torch.arange(size - kw.shape[3], size, device="cuda")
    sp = torch.arange(first, device="cuda")
    seen = torch.cat([qp - sp >= window, (kp >= 0) & (kp <= qp) & (qp - kp < window)], -1)
    sc = torch.cat([q @ ks.transpose(-1, -2), q @ kw.transpose(-1, -2)], -1).mul_(scale).masked_fill_(~seen, -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p /= total
    o = p[..., :first] @ vs + p[..., first:] @ vw
    whole = lambda t: t.reshape(b, h, blocks * size, -1)[:, :, :n]  # noqa: E731
    flat = lambda t: whole(t).transpose(1, 2).reshape(b * n, h * D)  # noqa: E731
    out = {"out": flat(o).to(s["qkv"].dtype), "lse": whole(top + total.log())[..., 0]}
    if not case["train"]:
        return out
    do = rows(s["dout"].float().view(b, n, h, D).transpose(1, 2))
    ds = torch.cat([do @ vs.transpose(-1, -2), do @ vw.transpose(-1, -2)], -1).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = ds[..., :first] @ ks + ds[..., first:] @ kw

    def keys(w, r):
        """Gradient of keys or values from the weights ``w`` of the rows ``r``: own block, the block after, first tokens."""
        t = w[..., first:].transpose(-1, -2) @ r
        own_block = t[:, :, :, -size:]
        if blocks > 1:
            own_block[:, :, :-1] += t[:, :, 1:, :-size]
        own_block = own_block.reshape(b, h, blocks * size, D)[:, :, :n]
        own_block[:, :, :first] += w[..., :first].flatten(2, 3).transpose(-1, -2) @ r.flatten(2, 3)
        return own_block.view(b, kv, g, n, D).sum(2).transpose(1, 2)[:, :, :, None]

    dq = whole(dq).transpose(1, 2).reshape(b, n, kv, g, D)
    out["dqkv"] = torch.cat([dq, keys(ds, q), keys(p, do)], 3).view(b * n, -1).to(s["qkv"].dtype)
    return out


def _plain_decode(s):
    case = s["case"]
    b, kv, g, first, window = case["batch"], case["kv"], case["group"], case["sinks"], case["window"]
    x, pos = s["qkv"].view(b, kv, g + 2, D), s["positions"]
    slot = torch.where(pos < first, pos, first + (pos - first) % window)
    rows = torch.arange(b, device="cuda")
    s["k"][rows, :, slot], s["v"][rows, :, slot] = x[:, :, g], x[:, :, g + 1]
    seen = torch.arange(first + window, device="cuda") <= pos[:, None]
    sc = (x[:, :, :g].float() @ s["k"].float().transpose(-1, -2) / math.sqrt(D)).masked_fill(~seen[:, None, None], -math.inf)
    e = (sc - sc.amax(-1, keepdim=True)).exp()
    out = (e / e.sum(-1, keepdim=True)) @ s["v"].float()
    return {"out": out.reshape(b, -1).to(s["qkv"].dtype), "k": s["k"], "v": s["v"]}


def _plain_distill(s):
    case = s["case"]
    vocab, t, w, scale = case["vocab"], case["temperature"], case["hard"], 1.0 / case["rows"]
    z = s["logits"][:, :vocab].float()
    there = (s["ids"] >= 0) & (s["ids"] < vocab)
    ids = torch.where(there, s["ids"], 0)
    lead = torch.where(there, s["values"].float(), -math.inf).amax(1, keepdim=True)
    e = torch.where(there, ((s["values"].float() - lead) / t).exp(), 0.0)
    total = e.sum(1, keepdim=True)
    some = (total > 0).float()
    p = e / torch.where(total > 0, total, 1.0)
    z = z - z.amax(1, keepdim=True)
    soft, hard = (z / t).exp(), z.exp()
    zs, zh = soft.sum(1, keepdim=True), hard.sum(1, keepdim=True)
    logp = torch.where(p > 0, p, 1.0).log()
    kl = (p * (logp - z.gather(1, ids) / t)).sum(1) + some[:, 0] * zs[:, 0].log()
    label = (s["targets"] >= 0) & (s["targets"] < vocab)
    y = torch.where(label, s["targets"], 0)[:, None]
    nll = torch.where(label, zh[:, 0].log() - z.gather(1, y)[:, 0], 0.0)
    loss = w * nll + (1 - w) * t * t * kl
    grad = torch.zeros(s["logits"].shape, device="cuda")
    grad[:, :vocab] = (1 - w) * t * some * (soft / zs) + w * label[:, None] * (hard / zh)
    grad.scatter_add_(1, ids, -(1 - w) * t * p)
    grad.scatter_add_(1, y, -w * label[:, None].float())
    return {"loss": loss, "grad": (grad * scale).to(s["logits"].dtype)}


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------
def _pairs(case):
    """(query, key) pairs of one head of one sequence."""
    n, w, s = case["seq"], min(case["window"] or case["seq"], case["seq"]), min(case["sinks"], case["seq"])
    total = w * (w + 1) // 2 + (n - w) * w
    far = max(0, n - w)                      # queries beyond the window: query w - 1 + i sees min(i, s) first tokens outside it
    return total + sum(min(i, s) for i in range(1, min(far, s) + 1)) + max(0, far - s) * s


def work(case):
    k = case["kind"]
    if k == "rotary":
        t = case["batch"] * case["seq"]
        pairs = t * case["kv"] * (case["group"] + 1) * case["rot"] // 2
        return {"bytes": 4 * t * _width(case) + (8 * t if case["far"] else 0), "flops": 6 * pairs}
    if k == "window":
        t, h = case["batch"] * case["seq"], case["kv"] * case["group"]
        forward = 4 * D * _pairs(case) * case["batch"] * h
        b = 2 * t * _width(case) + 2 * t * h * D + 4 * t * h
        if case["train"]:
            return {"bytes": 2 * b - 4 * t * h + 2 * t * h * D, "flops": forward * 3.5}
        return {"bytes": b, "flops": forward}
    if k == "decode":
        seen = sum(min(p + 1, case["sinks"] + case["window"]) for p in _stops(case))
        b, h = case["batch"], case["kv"] * case["group"]
        return {"bytes": 4 * seen * case["kv"] * D + 2 * b * _width(case) + 2 * b * h * D + 8 * b + 4 * b * case["kv"] * D,
                "flops": 4 * seen * h * D}
    rows, padded = case["rows"], -(-case["vocab"] // VOCAB_PAD) * VOCAB_PAD
    return {"bytes": rows * (2 * case["vocab"] + 2 * padded + 12 * case["top"] + 8 + 4), "flops": 8 * rows * case["vocab"]}


def _cost(case):
    """Operations, or those for which the card would have time while it moves the bytes."""
    w = work(case)
    return max(w["flops"], 250 * w["bytes"])


# ----------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotary": _exact_rotary, "window": _exact_window, "decode": _exact_decode, "distill": _exact_distill}[case["kind"]](case, s)


def _exact_rotary(case, s):
    """Every pair of features is a complex number that is multiplied by m exp(i position frequency)."""
    rot, base, factor = case["rot"], 10000.0, case["factor"]
    freq, m = [], 1.0
    if case["scaling"] == "by_parts":
        m = 1.0 + 0.1 * math.log(factor)
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if case["scaling"] == "base":
            f = (base * factor ** (rot / (rot - 2.0))) ** (-2.0 * i / rot)
        elif case["scaling"] == "linear":
            f = f / factor
        elif case["scaling"] == "by_parts":
            share = min(1.0, max(0.0, (8192 * f / (2 * math.pi) - 1.0) / 31.0))
            f = share * f + (1.0 - share) * f / factor
        freq.append(f)
    tokens = case["batch"] * case["seq"]
    pos = s["positions"] if case["far"] else torch.arange(case["seq"], device="cuda").repeat(case["batch"])
    angle = pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, m), -angle if case["inverse"] else angle)[:, None, None]
    x = s["x"].double().view(tokens, case["kv"], case["group"] + 2, D)
    qk = x[:, :, :-1, :rot]
    if case["layout"] == "half":
        z = torch.complex(qk[..., :rot // 2].contiguous(), qk[..., rot // 2:].contiguous()) * turn
        x[:, :, :-1, :rot] = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.complex(qk[..., 0::2].contiguous(), qk[..., 1::2].contiguous()) * turn
        x[:, :, :-1, :rot] = torch.stack([z.real, z.imag], -1).flatten(-2)
    return x.view(tokens, -1)


def _exact_window(case, s):
    """Head by head over the whole matrix of scores."""
    b, n, kv, g = case["batch"], case["seq"], case["kv"], case["group"]
    if b * kv * g * n * n > 2 ** 33:
        return None
    w, first = case["window"] or n, case["sinks"]
    x = s["qkv"].view(b, n, kv, g + 2, D)
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
    hidden = (j > i) | ((i - j >= w) & (j >= first))
    out = torch.empty(b, n, kv, g, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(b, kv, g, n, dtype=torch.float64, device="cuda")
    grad = torch.zeros(b, n, kv, g + 2, D, dtype=torch.float64, device="cuda")
    for bi in range(b):
        for hi in range(kv):
            k, v = x[bi, :, hi, g].double(), x[bi, :, hi, g + 1].double()
            for qi in range(g):
                q = x[bi, :, hi, qi].double()
                sc = ((q @ k.T) / math.sqrt(D)).masked_fill_(hidden, -math.inf)
                lse[bi, hi, qi] = torch.logsumexp(sc, 1)
                p = torch.softmax(sc, 1)
                out[bi, :, hi, qi] = p @ v
                if case["train"]:
                    do = s["dout"].view(b, n, kv, g, D)[bi, :, hi, qi].double()
                    dp = do @ v.T
                    ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(D)
                    grad[bi, :, hi, qi] = ds @ k
                    grad[bi, :, hi, g] += ds.T @ q
                    grad[bi, :, hi, g + 1] += p.T @ do
    got = {"out": out.view(b * n, -1), "lse": lse.view(b, kv * g, n)}
    if case["train"]:
        got["dqkv"] = grad.view(b * n, -1)
    return got


def _exact_decode(case, s):
    """Sequence by sequence over the slots that hold a position."""
    g, first, window = case["group"], case["sinks"], case["window"]
    k, v = s["k"].double(), s["v"].double()
    out = torch.empty(case["batch"], case["kv"], g, D, dtype=torch.float64, device="cuda")
    for i, p in enumerate(s["positions"].tolist()):
        x = s["qkv"][i].double().view(case["kv"], g + 2, D)
        slot = p if p < first else first + (p - first) % window
        k[i, :, slot], v[i, :, slot] = x[:, g], x[:, g + 1]
        held = min(p + 1, first + window)
        weights = torch.softmax(torch.einsum("hgd,hnd->hgn", x[:, :g], k[i, :, :held]) / math.sqrt(D), -1)
        out[i] = torch.einsum("hgn,hnd->hgd", weights, v[i, :, :held])
    return {"out": out.view(case["batch"], -1), "k": k, "v": v}


def _exact_distill(case, s):
    """The gradient by its definition: of the dense teacher distribution and of the one-hot label."""
    vocab, t, w = case["vocab"], case["temperature"], case["hard"]
    rows = case["rows"]
    z = s["logits"][:, :vocab].double()
    there = (s["ids"] >= 0) & (s["ids"] < vocab)
    kept = torch.full((rows, vocab), -math.inf, dtype=torch.float64, device="cuda")
    r, c = there.nonzero(as_tuple=True)
    kept[r, s["ids"][r, c]] = s["values"][r, c].double()
    some = there.any(1)
    target = torch.zeros_like(kept)
    target[some] = torch.softmax(kept[some] / t, 1)
    del kept
    logq = torch.log_softmax(z / t, 1)
    kl = torch.where(target > 0, target * (target.clamp_min(1e-300).log() - logq), 0.0).sum(1)
    g = (1 - w) * t * (logq.exp() * some[:, None] - target)
    del target, logq
    logq = torch.log_softmax(z, 1)
    label = ((s["targets"] >= 0) & (s["targets"] < vocab)).nonzero()[:, 0]
    nll = torch.zeros(rows, dtype=torch.float64, device="cuda")
    nll[label] = -logq[label, s["targets"][label]]
    hard = torch.zeros_like(z)
    hard[label] = logq[label].exp()
    hard[label, s["targets"][label]] -= 1
    grad = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    grad[:, :vocab] = (g + w * hard) / rows
    return {"loss": w * nll + (1 - w) * t * t * kl, "grad": grad}
