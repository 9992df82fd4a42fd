"""A windowed GPT with rotary positions and shared heads: training on emulated meshes against a dense model, distillation, token by token."""
import math

import pytest
import torch

from meshslice_b200.models.decode import GPTDecoder
from meshslice_b200.models.gpt import DistillTargets, GPTConfig, GPTModel
from meshslice_b200.ops import functional as F
from meshslice_b200.ops.rotary import Rotary, RotaryConfig
from meshslice_b200.parallel.mesh import EmuMesh, ShardedTensor
from meshslice_b200.trainer import param_elems

ROT = RotaryConfig(head_dim=16, rot_dim=16, layout="interleaved", scaling="by_parts", factor=4.0, original_len=16)
CFG = GPTConfig(n_layers=2, d_model=128, n_heads=8, kv_heads=4, ffn=256, vocab=500, seq=37, ksplits=(2, 2, 2, 2), head_ksplit=2,
                vocab_pad=256, dtype=torch.float32, window=9, sinks=2, rotary=ROT)


def _cols(mesh, st):
    return torch.cat([st.shards[(0, c)] for c in range(mesh.C)], dim=-1)


def _dense_logits(model, mesh, cfg, ids, leaf):
    """Plain forward of the same network; ``ids`` [batch, n]."""
    B, n = ids.shape
    kv, g, D = cfg.kv_heads, cfg.n_heads // cfg.kv_heads, cfg.d_model // cfg.n_heads
    x = leaf("tok", _cols(mesh, model.tok))[ids.reshape(-1)]
    ln = lambda v, l, t: torch.nn.functional.layer_norm(v, (cfg.d_model,), leaf(t + ".g", _cols(mesh, l.gamma)), leaf(t + ".b", _cols(mesh, l.bias)), cfg.eps)

    def lin(v, layer, t):
        w = leaf(t, mesh.unshard(layer.weight))
        return v @ (w.t() if layer.dataflow == "ls" else w)
    cos, sin = Rotary(cfg.rotary).cos_sin(torch.arange(n))
    i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
    hidden = (j > i) | ((i - j >= cfg.window) & (j >= cfg.sinks))
    for b, blk in enumerate(model.blocks):
        qkv = lin(ln(x, blk.ln1, f"{b}.ln1"), blk.in_proj, f"{b}.in").view(B, n, kv, g + 2, D)
        c, s = cos[:, None, None], sin[:, None, None]
        u, v = qkv[..., 0::2], qkv[..., 1::2]
        turned = torch.stack([u * c - v * s, v * c + u * s], -1).flatten(-2)
        q, k, v = turned[:, :, :, :g], turned[:, :, :, g], qkv[:, :, :, g + 1]
        sc = torch.einsum("bnhgd,bmhd->bhgnm", q, k) / math.sqrt(D)
        a = torch.einsum("bhgnm,bmhd->bnhgd", torch.softmax(sc.masked_fill(hidden, -math.inf), -1), v).reshape(B * n, -1)
        x = x + lin(a, blk.out_proj, f"{b}.out")
        m = torch.nn.functional.gelu(lin(ln(x, blk.ln2, f"{b}.ln2"), blk.ff1, f"{b}.ff1"), approximate="tanh")
        x = x + lin(m, blk.ff2, f"{b}.ff2")
    return lin(ln(x, model.ln_f, "lnf"), model.head, "head")[:, :cfg.vocab]


@pytest.mark.parametrize("distill", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (2, 2), (1, 4)])
def test_loss_and_gradients_match_dense_model(shape, distill):
    R, C = shape
    mesh = EmuMesh(R, C)
    model, B, n, K, T, w = GPTModel(mesh, CFG), 4, CFG.seq, 5, 2.0, 0.25
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, CFG.vocab, (B, n + 1), generator=gen)
    tid = torch.stack([torch.randperm(CFG.vocab, generator=gen)[:K] for _ in range(B * n)])
    tval = torch.randn(B * n, K, generator=gen)
    per = B // R
    rows = lambda t: ShardedTensor(mesh, {(r, c): t[r * per * n:(r + 1) * per * n].clone() for (r, c) in mesh.coords()})
    teacher = DistillTargets(rows(tid), rows(tval), T, w) if distill else None
    tok, tgt = ids[:, :-1].reshape(-1), ids[:, 1:].reshape(-1)
    loss = model.forward_backward(rows(tok), rows(tgt), B * n, teacher)
    model.sync_replicated_grads()
    P = {}

    def leaf(name, t):
        P[name] = t.clone().float().requires_grad_(True)
        return P[name]
    z = _dense_logits(model, mesh, CFG, ids[:, :-1], leaf)
    want = torch.nn.functional.cross_entropy(z, tgt)
    if distill:
        p = torch.softmax(tval / T, 1)
        kl = (p * (p.log() - torch.log_softmax(z / T, 1).gather(1, tid))).sum(1).mean()
        want = w * want + (1 - w) * T * T * kl
    want.backward()
    assert abs(sum(loss.shards[(r, 0)] for r in range(R)).item() - want.item()) < 1e-4
    b0 = model.blocks[0]
    for layer, tag in ((b0.in_proj, "0.in"), (b0.out_proj, "0.out"), (b0.ff1, "0.ff1"), (model.blocks[1].in_proj, "1.in"), (model.head, "head")):
        assert torch.allclose(mesh.unshard(layer.grad), P[tag].grad, atol=2e-5, rtol=1e-3), tag
    assert torch.allclose(_cols(mesh, model.dtok), P["tok"].grad, atol=2e-5, rtol=1e-3)


def test_parameters_and_sizes():
    """Rotary models have no learned positions; buffers and counts follow the shared heads."""
    mesh = EmuMesh(1, 1)
    model = GPTModel(mesh, CFG)
    params = model.parameters()
    assert model.pos is None and "pos" not in [n for n, *_ in params]
    total = sum(p.shards[(0, 0)].numel() for _, p, _, _ in params)
    assert total == CFG.n_params()
    sharded, rep = param_elems(CFG, 1, 1)
    pad = lambda v: (v + 127) // 128 * 128
    for kind, n in (("sharded", sharded), ("row_replicated", rep)):
        assert n == sum(pad(p.shards[(0, 0)].numel()) for _, p, _, k in params if k == kind)
    for bad in (dict(kv_heads=3), dict(window=-1), dict(causal=False), dict(rotary=RotaryConfig(head_dim=32))):
        with pytest.raises(ValueError):
            GPTConfig(**{**dict(n_layers=1, d_model=128, n_heads=8, window=4), **bad})
    with pytest.raises(ValueError):
        GPTModel(EmuMesh(1, 8), CFG)


@pytest.mark.parametrize("prompt", [1, 8, 30])
@pytest.mark.parametrize("rotary", [ROT, None])
def test_token_by_token_is_the_whole_sequence(rotary, prompt):
    cfg = GPTConfig(**{**CFG.__dict__, "rotary": rotary})
    mesh = EmuMesh(1, 1)
    model = GPTModel(mesh, cfg)
    ids = torch.randint(0, cfg.vocab, (2, cfg.seq), generator=torch.Generator().manual_seed(2))
    want = model.forward(ShardedTensor(mesh, {(0, 0): ids.reshape(-1)})).shards[(0, 0)][:, :cfg.vocab].view(2, cfg.seq, -1)
    d = GPTDecoder(model, 2)
    got = [d.prefill(ids[:, :prompt])]
    got += [d.step(ids[:, p], torch.full((2,), p)) for p in range(prompt, cfg.seq)]
    assert torch.allclose(torch.stack(got, 1), want[:, prompt - 1:], atol=1e-4, rtol=1e-4)
    with pytest.raises(ValueError):
        d.step(ids[:1, 0], torch.zeros(2))
    with pytest.raises(ValueError):
        GPTDecoder(GPTModel(mesh, GPTConfig(**{**cfg.__dict__, "window": 0})), 2)


# ---------------------------------------------------------------------------------------------- on a GPU
@pytest.mark.gpu
def test_example_runs_and_learns():
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "bench" / "distill_window.py"
    spec = importlib.util.spec_from_file_location("distill_window", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses, written = mod.main(["--steps", "12", "--seqlen", "333", "--window", "64", "--scale-factor", "2"])
    assert losses[-1] < losses[0] and all(math.isfinite(v) for v in losses)
    assert len(written) == 4 and all(0 <= t < 1000 for row in written for t in row)


@pytest.mark.gpu
def test_decoding_on_a_gpu_is_the_whole_sequence():
    """Logits of 32 tokens written one by one against those of the whole sequence: both paths round activations to bf16 at the same
    places, but sum in different orders, so the streams differ by the rounding of each block's outputs: 2 blocks and the head, each
    2^-8 of values of the residual stream's size, whose effect on the logits is bounded by their own size."""
    from meshslice_b200 import _native
    from meshslice_b200.parallel.engine import LocalGemmEngine
    mesh = EmuMesh(1, 1)
    LocalGemmEngine(mesh)
    cfg = GPTConfig(n_layers=2, d_model=512, n_heads=4, kv_heads=2, ffn=1024, vocab=777, seq=200, vocab_pad=256, window=50, sinks=3,
                    rotary=RotaryConfig(), init_std=0.05)
    model = GPTModel(mesh, cfg, device=torch.device("cuda", 0))
    ids = torch.randint(0, cfg.vocab, (3, cfg.seq), generator=torch.Generator().manual_seed(2)).cuda()
    want = model.forward(ShardedTensor(mesh, {(0, 0): ids.reshape(-1)})).shards[(0, 0)][:, :cfg.vocab].view(3, cfg.seq, -1).float()
    d = GPTDecoder(model, 3)
    got = [d.prefill(ids[:, :169])] + [d.step(ids[:, p], torch.full((3,), p, device="cuda")) for p in range(169, cfg.seq)]
    _native.check_status()
    diff = torch.stack(got, 1).float() - want[:, 168:]
    assert diff.norm() < 6 * 2.0 ** -8 * want[:, 168:].norm()


def test_operations_of_a_window():
    """Attention's share of the operations counts the pairs that a window and its first tokens leave."""
    base = dict(n_layers=3, d_model=128, n_heads=8, ffn=256, vocab=500, vocab_pad=256)
    for seq, window, sinks in ((50, 7, 0), (50, 7, 3), (64, 60, 30), (40, 1, 1)):
        pairs = sum(1 for i in range(seq) for j in range(i + 1) if i - j < window or j < sinks)
        rest = GPTConfig(**base, seq=seq).flops_per_token() - 3 * 4 * seq * 128 * 3 * 0.5
        got = GPTConfig(**base, seq=seq, window=window, sinks=sinks).flops_per_token() - rest
        assert abs(got - 3 * 4 * 128 * 3 * pairs / seq) < 1e-6 * got


@pytest.mark.parametrize("rotary", [ROT, None])
def test_decoder_refuses_tokens_and_positions_that_it_has_nothing_for(rotary):
    """Types, devices, ids outside the vocabulary, prompts and positions beyond the learned ones (of which decoding with a cache of fixed
    size is free otherwise)."""
    cfg = GPTConfig(**{**CFG.__dict__, "rotary": rotary, "seq": 12})
    model = GPTModel(EmuMesh(1, 1), cfg)
    d = GPTDecoder(model, 2)
    ids = torch.randint(0, cfg.vocab, (2, 20), generator=torch.Generator().manual_seed(3))
    at = lambda p: torch.full((2,), p)
    if rotary is None:
        for call in (lambda: d.prefill(ids[:, :13]), lambda: d.step(ids[:, 0], at(12)), lambda: d.step(ids[:, 0], torch.tensor([1, 400]))):
            with pytest.raises(ValueError):
                call()
    else:
        assert d.prefill(ids[:, :13]).isfinite().all() and d.step(ids[:, 13], at(13)).isfinite().all()
    d.prefill(ids[:, :11])
    for tokens, positions in ((ids[:, 11].int(), at(11)), (ids[:, 11], at(11).int()), (ids[:, 11], at(11).float()), (ids[:, 11].float(), at(11)),
                              (ids[:, 11].to("meta"), at(11)), (ids[:, 11], at(11).to("meta")), (torch.tensor([0, -1]), at(11)),
                              (torch.tensor([cfg.vocab_padded, 0]), at(11))):
        with pytest.raises(ValueError):
            d.step(tokens, positions)
    for prompts in (ids[:, :5].int(), ids[:, :5].float(), ids[:, :5].to("meta"), ids[:, :5] - cfg.vocab):
        with pytest.raises(ValueError):
            d.prefill(prompts)
    want = d.step(ids[:, 11], at(11))
    d.prefill(ids[:, :11])
    got = d.step(torch.tensor([int(ids[0, 11]), -1]), torch.tensor([11, -1]))          # an idle sequence's token is not looked at
    assert torch.equal(got[0], want[0])


@pytest.mark.gpu
def test_decoder_on_a_gpu_reads_nothing_outside_its_tables():
    """Ids outside the vocabulary count as the nearest one; positions without a learned vector show as NaN in their own sequence."""
    from meshslice_b200 import _native
    from meshslice_b200.parallel.engine import LocalGemmEngine
    mesh = EmuMesh(1, 1)
    LocalGemmEngine(mesh)
    for rotary in (RotaryConfig(), None):
        cfg = GPTConfig(n_layers=1, d_model=256, n_heads=2, ffn=512, vocab=250, seq=40, vocab_pad=256, window=16, rotary=rotary)
        model = GPTModel(mesh, cfg, device=torch.device("cuda", 0))
        d = GPTDecoder(model, 3)
        ids = torch.randint(0, cfg.vocab, (3, 41), generator=torch.Generator().manual_seed(4)).cuda()
        with pytest.raises(ValueError):
            d.step(ids[:, 0].int(), ids[:, 0])
        with pytest.raises(ValueError):
            d.step(ids[:, 0], ids[:, 0].cpu())
        if rotary is None:
            with pytest.raises(ValueError):
                d.prefill(ids)
        d.prefill(ids[:, :39])
        want = d.step(ids[:, 39], torch.tensor([39, 39, -1], device="cuda"))
        d.prefill(ids[:, :39])
        tokens = ids[:, 39].clone()
        tokens[2] = -(1 << 40)
        got = d.step(tokens, torch.tensor([39, 1 << 20, -1], device="cuda"))
        assert torch.equal(got[0], want[0]) and bool(got[1].isnan().all()) == (rotary is None)
        d.prefill(ids[:, :39])
        tokens[1], tokens[0] = 1 << 40, cfg.vocab_padded - 1
        same = d.step(tokens, torch.full((3,), 39, device="cuda"))
        assert same[1].isfinite().all() and same[0].isfinite().all()
    _native.check_status()


def _held(model):
    """What the layers hold for a backward pass, by identity."""
    layers = [l for b in model.blocks for l in (*b.layers(), b.attn, b.gelu)] + [model.ln_f, model.head]
    return [(type(l).__name__, getattr(l, "_x", None), getattr(l, "_saved", None)) for l in layers]


@pytest.mark.parametrize("change", [{}, dict(rotary=None), dict(window=0, kv_heads=0, sinks=0, rotary=None)])
def test_teacher_and_decoder_hold_nothing_and_disturb_nothing(change):
    """Without a backward pass to come no activation is held; what a forward pass holds is there when the decoder or a teacher's logits
    were asked for in between, and its gradients are the same."""
    cfg = GPTConfig(**{**CFG.__dict__, **change})
    mesh = EmuMesh(1, 1)
    model = GPTModel(mesh, cfg)
    gen = torch.Generator().manual_seed(5)
    ids = torch.randint(0, cfg.vocab, (2 * cfg.seq,), generator=gen)
    tokens = ShardedTensor(mesh, {(0, 0): ids})

    def between():
        model.top_logits(tokens, 3)
        if cfg.window:
            d = GPTDecoder(model, 2)
            d.prefill(ids.view(2, -1)[:, :4])
            d.step(ids[:2], torch.full((2,), 4))
    between()
    assert all(x is None and saved is None for _, x, saved in _held(model))
    assert all(l.h is None for b in model.blocks for l in (b.ln1, b.ln2)) and model.ln_f.h is None

    block = model.blocks[0]
    x, dh, dm = (torch.randn(2 * cfg.seq, cfg.d_model, generator=gen) for _ in range(3))
    grads = []
    for disturb in (False, True):
        model.zero_grad()
        st = lambda t: ShardedTensor(mesh, {(0, 0): t.clone()})
        h, _ = block.forward(st(x), None)
        held, residual = _held(model), h.shards[(0, 0)].clone()
        assert any(v is not None for _, v, _ in held)
        if disturb:
            between()
            assert all(a[1] is b[1] and a[2] is b[2] for a, b in zip(held, _held(model)))
            assert torch.equal(h.shards[(0, 0)], residual)
        dx, _ = block.backward(st(dh), st(dm))
        grads.append([dx.shards[(0, 0)]] + [g.shards[(0, 0)].clone() for _, _, g, _ in model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_counts_without_shared_heads_are_those_of_three_widths():
    """The input projection of a model whose heads each have a key and a value is three widths wide, whether or not the heads divide it
    (counts are asked of sizes that no device has run yet)."""
    for d, heads in ((128, 8), (100, 8), (1000, 3), (12, 24)):
        cfg = GPTConfig(n_layers=2, d_model=d, n_heads=heads, ffn=4 * d, vocab=500, seq=64, vocab_pad=256)
        per_layer = 3 * d * d + d * d + 2 * d * 4 * d + 4 * d
        assert cfg.n_params() == 2 * per_layer + (512 + 64) * d + d * 512 + 2 * d
        assert cfg.flops_per_token() == 3.0 * (2 * (3 * d * d + d * d + 8 * d * d) * 2 + 2 * d * 512 + 4 * 64 * d * 2 * 0.5)
    assert GPTConfig(n_layers=1, d_model=128, n_heads=8, kv_heads=8).qkv_dim == 384
    assert GPTConfig(n_layers=1, d_model=128, n_heads=8, kv_heads=2).qkv_dim == 192
