"""A decoder with gated feed-forward blocks, the head's loss without logits and orthogonal updates: on emulated meshes against a dense
model, on a GPU against the framework's other paths, and all of it together."""
import math

import pytest
import torch

from meshslice_b200.checkpoint import load_checkpoint, save_checkpoint
from meshslice_b200.models.decode import GPTDecoder
from meshslice_b200.models.gpt import GPTConfig, GPTModel
from meshslice_b200.models.sharded_layers import ShardedGatedFF
from meshslice_b200.ops import functional as F
from meshslice_b200.ops.orthogonal import COEFFICIENTS
from meshslice_b200.optim import AdamW, FlatGroup, Muon
from meshslice_b200.parallel.mesh import EmuMesh, ShardedTensor
from meshslice_b200.trainer import Trainer, TrainConfig, param_elems

gpu = pytest.mark.gpu
CFG = dict(n_layers=2, d_model=64, n_heads=4, ffn=128, vocab=200, seq=12, ksplits=(2, 2, 2, 2), head_ksplit=2, vocab_pad=64, dtype=torch.float32)


def dense_loss(model, mesh, cfg, tok, tgt, leaf):
    n, D = cfg.seq, cfg.d_model // cfg.n_heads
    cols = lambda st: torch.cat([st.shards[(0, c)] for c in range(mesh.C)], dim=-1)
    B = tok.numel() // n
    x = leaf("tok", cols(model.tok))[tok] + leaf("pos", cols(model.pos)).repeat(B, 1)
    ln = lambda v, l, t: torch.nn.functional.layer_norm(v, (cfg.d_model,), leaf(t + ".g", cols(l.gamma)), leaf(t + ".b", cols(l.bias)), cfg.eps)

    def lin(v, layer, t):
        w = leaf(t, mesh.unshard(layer.weight))
        return v @ (w.t() if layer.dataflow == "ls" else w)
    act = torch.nn.functional.silu if cfg.gated == "silu" else lambda v: torch.nn.functional.gelu(v, approximate="tanh")
    for i, b in enumerate(model.blocks):
        q, k, v = lin(ln(x, b.ln1, f"{i}.ln1"), b.in_proj, f"{i}.in").view(B, n, cfg.n_heads, 3, D).unbind(3)
        s = torch.einsum("bnhd,bmhd->bhnm", q, k) / math.sqrt(D)
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
        a = torch.einsum("bhnm,bmhd->bnhd", torch.softmax(s, -1), v).reshape(B * n, -1)
        x = x + lin(a, b.out_proj, f"{i}.out")
        y = ln(x, b.ln2, f"{i}.ln2")
        x = x + lin(act(lin(y, b.ff.gate, f"{i}.gate")) * lin(y, b.ff.up, f"{i}.up"), b.ff.down, f"{i}.down")
    z = lin(ln(x, model.ln_f, "lnf"), model.head, "head")[:, :cfg.vocab]
    return torch.nn.functional.cross_entropy(z, tgt)


@pytest.mark.parametrize("shape,act,dataflows,head_rows", [
    ((1, 1), "silu", ("os", "os", "os", "ls"), 5), ((1, 1), "gelu", ("os", "ls", "ls", "os"), 0), ((1, 1), "silu", ("os", "os", "os", "ls"), None),
    ((2, 2), "silu", ("os", "os", "os", "ls"), None), ((1, 4), "gelu", ("ls", "os", "ls", "os"), None)])
def test_loss_and_gradients_match_a_dense_model(shape, act, dataflows, head_rows):
    R, C = shape
    mesh, cfg = EmuMesh(R, C), GPTConfig(**CFG, gated=act, dataflows=dataflows, head_rows=head_rows)
    model, B = GPTModel(mesh, cfg), 2 * R
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, cfg.vocab, (B, cfg.seq + 1), generator=gen)
    tok, tgt = ids[:, :-1].reshape(-1), ids[:, 1:].reshape(-1)
    per = B // R * cfg.seq
    rows = lambda t: ShardedTensor(mesh, {(r, c): t[r * per:(r + 1) * per].clone() for (r, c) in mesh.coords()})
    loss = model.forward_backward(rows(tok), rows(tgt), tok.numel())
    model.sync_replicated_grads()
    P = {}

    def leaf(name, t):
        P[name] = t.clone().float().requires_grad_(True)
        return P[name]
    want = dense_loss(model, mesh, cfg, tok, tgt, leaf)
    want.backward()
    assert abs(sum(loss.shards[(r, 0)] for r in range(R)).item() - want.item()) < 1e-4
    for i, b in enumerate(model.blocks):
        for layer, t in ((b.in_proj, "in"), (b.out_proj, "out"), (b.ff.gate, "gate"), (b.ff.up, "up"), (b.ff.down, "down")):
            assert torch.allclose(mesh.unshard(layer.grad), P[f"{i}.{t}"].grad, rtol=1e-3, atol=1e-6), (i, t)
    assert torch.allclose(mesh.unshard(model.head.grad), P["head"].grad, rtol=1e-3, atol=1e-6)
    assert torch.allclose(torch.cat([model.dtok.shards[(0, c)] for c in range(C)], 1), P["tok"].grad, rtol=1e-3, atol=1e-6)
    if (R, C) == (1, 1):
        losses = model.token_losses(rows(tok), rows(tgt)).local()
        assert losses.shape == tok.shape and abs(losses.mean().item() - want.item()) < 1e-4


def test_sizes_and_names():
    cfg = GPTConfig(**CFG, gated="silu")
    model = GPTModel(EmuMesh(1, 1), cfg)
    weights = sum(p.local().numel() for n, p, _, _ in model.parameters() if n not in ("tok", "pos"))
    assert cfg.n_params() == weights + model.tok.local().numel() + model.pos.local().numel()
    sharded, _ = param_elems(cfg, 1, 1)
    pad = lambda n: -(-n // 128) * 128
    assert sharded == sum(pad(p.local().numel()) for _, p, _, kind in model.parameters() if kind == "sharded")
    assert cfg.flops_per_token() > GPTConfig(**CFG).flops_per_token()
    assert len({n for n, _, _, _ in model.parameters()}) == len(model.parameters())
    assert len(model.blocks[0].matrices()) == 5


def test_refusals():
    with pytest.raises(ValueError):
        GPTConfig(**CFG, gated="relu")
    with pytest.raises(ValueError):
        GPTConfig(**CFG, gated="silu", dataflows=("os", "os", "rs", "ls"))
    with pytest.raises(ValueError):
        GPTConfig(**CFG, head_rows=-1)
    with pytest.raises(ValueError):
        GPTModel(EmuMesh(1, 2), GPTConfig(**CFG, head_rows=0))
    with pytest.raises(ValueError):
        GPTModel(EmuMesh(1, 2), GPTConfig(**CFG)).token_losses(None, None)
    with pytest.raises(ValueError):
        ShardedGatedFF(EmuMesh(1, 1), "meshslice", ("os", "rs"), (1, 1), 64, 96)
    with pytest.raises(ValueError):
        ShardedGatedFF(EmuMesh(1, 1), "meshslice", ("os", "os"), (1, 1), 64, 96, "tanh")
    for kw in (dict(optimizer="sgd"), dict(optimizer="muon")):
        with pytest.raises(ValueError):
            Trainer(GPTConfig(**CFG), TrainConfig(global_batch=2, micro_batch=1, **kw), mesh_shape=(1, 2), device=torch.device("cpu"))


def test_decoder_answers_as_the_model():
    cfg = GPTConfig(**CFG, gated="gelu", window=8, sinks=1)
    model = GPTModel(EmuMesh(1, 1), cfg)
    ids = torch.randint(0, cfg.vocab, (2, cfg.seq), generator=torch.Generator().manual_seed(0))
    want = model.forward(ShardedTensor(model.mesh, {(0, 0): ids.reshape(-1)}), keep=False).local()[:, :cfg.vocab].view(2, cfg.seq, -1)
    dec = GPTDecoder(model, 2)
    got = [dec.prefill(ids[:, :5])] + [dec.step(ids[:, i], torch.full((2,), i)) for i in range(5, cfg.seq)]
    assert torch.allclose(torch.stack(got, 1), want[:, 4:], atol=1e-4)


# ----------------------------------------------------------------------------------------------
# Muon
# ----------------------------------------------------------------------------------------------
def flat(device, seed=0, dtype=torch.float32, grad_dtype=torch.float32):
    """A group with three matrices of one shape at equal distances, one of another shape, and elements around them."""
    gen = torch.Generator().manual_seed(seed)
    r = lambda n: torch.randn(n, generator=gen)
    sizes = [128, 24 * 40, 128, 24 * 40, 128, 24 * 40, 64, 64 * 16, 32]
    param, grad = r(sum(sizes)).to(dtype).to(device), r(sum(sizes)).to(grad_dtype).to(device)
    at = [sum(sizes[:i]) for i in range(len(sizes))]
    view = lambda t, i, *s: t[at[i]:at[i] + sizes[i]].view(*s)
    matrices = lambda t: [view(t, 1, 24, 40), view(t, 3, 24, 40), view(t, 5, 24, 40), view(t, 7, 64, 16)]
    rest = [(0, 128), (at[2], at[3]), (at[4], at[5]), (at[6], at[7]), (at[8], at[8] + 32)]
    return FlatGroup(param, grad, "sharded"), matrices, rest


def polynomial(u):
    x = u.double()
    x = x.mT if x.shape[0] > x.shape[1] else x
    x = x / x.norm()
    a, b, c = COEFFICIENTS
    for _ in range(5):
        q = x @ x.T
        x = a * x + (b * q + c * q @ q) @ x
    return x.mT if u.shape[0] > u.shape[1] else x


def two_steps(device, nesterov, dtype, grad_dtype, off):
    group, matrices, rest = flat(device, dtype=dtype, grad_dtype=grad_dtype)
    other = FlatGroup(torch.ones(64, device=device, dtype=dtype), torch.ones(64, device=device), "row_replicated")
    opt = Muon([group, other], matrices(group.param), nesterov=nesterov, momentum=0.9, lr=0.02, weight_decay=0.1, max_grad_norm=1.0)
    assert sorted(s[1:] for s in opt._stacks) == [(128, 24 * 40 + 128, 3, 24, 40), (128 * 3 + 24 * 40 * 3 + 64, 64 * 16, 1, 64, 16)]
    plain = AdamW([FlatGroup(group.param.clone(), group.grad, "sharded"), FlatGroup(other.param.clone(), other.grad, "row_replicated")], lr=0.02,
                  weight_decay=0.1, max_grad_norm=1.0)
    masters = [t.double().cpu().clone() for t in matrices(group.master)]
    momentum = [torch.zeros_like(t) for t in masters]
    for _ in range(2):
        opt.step()
        plain.step()
        scale = min(1.0, 1.0 / (float(plain.last_grad_norm) + 1e-6))
        for i, g in enumerate(matrices(group.grad)):
            g = g.double().cpu() * scale
            momentum[i] = 0.9 * momentum[i] + g
            u = g + 0.9 * momentum[i] if nesterov else momentum[i]
            masters[i] = masters[i] - 0.02 * (0.2 * math.sqrt(max(g.shape)) * polynomial(u) + 0.1 * masters[i])
        group.grad.mul_(-0.5)
    for got, m, master, mom in zip(matrices(group.master), matrices(group.m), masters, momentum):
        assert (m.double().cpu() - mom).norm() < 1e-5 * mom.norm()
        # of two updates of 0.02 * 0.2 sqrt(max) O, whose norm is about sqrt(min)
        assert (got.double().cpu() - master).norm() < off * 2 * 0.004 * math.sqrt(max(got.shape) * min(got.shape)) + 2.0 ** -22 * master.norm()
    assert torch.equal(group.param, group.master.to(dtype))
    # the gradients' norm is summed in any order: some 2^-22 of it, and of m; steps of at most lr
    same = lambda x, y: ((x - y).abs() <= 2.0 ** -21 * (y.abs() + 0.02)).all()
    for a, b in rest:
        assert same(group.master[a:b], plain.groups[0].master[a:b]) and same(group.m[a:b], plain.groups[0].m[a:b])
    assert same(other.master, plain.groups[1].master)
    assert all(v.count_nonzero() == 0 for v in matrices(group.v))


@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_cpu(nesterov):
    two_steps("cpu", nesterov, torch.float32, torch.float32, 1e-5)


@gpu
@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
def test_muon_gpu(nesterov, grad_dtype, monkeypatch):
    """fp16 factors: some 1e-3 of the update (the operator's own tests say how much); in one stack and with one matrix at a time."""
    from meshslice_b200 import optim
    two_steps("cuda", nesterov, torch.bfloat16, grad_dtype, 1e-2)
    monkeypatch.setattr(optim, "UPDATE_BYTES", 5000)
    two_steps("cuda", nesterov, torch.bfloat16, grad_dtype, 1e-2)


def test_muon_refusals():
    group, matrices, _ = flat("cpu")
    for bad in ([group.param[:1000].view(10, 100)] + [group.param[500:600].view(10, 10)], [torch.zeros(8, 8)], [group.param[2:66].view(8, 8)],
                [group.param[:9].view(3, 3)], [group.param[:64]]):
        with pytest.raises(ValueError):
            Muon([group], bad)
    with pytest.raises(ValueError):
        Muon([group], matrices(group.param), momentum=1.0)
    with pytest.raises(ValueError):
        Muon([group], matrices(group.param), mesh=EmuMesh(1, 2))


# ----------------------------------------------------------------------------------------------
# together
# ----------------------------------------------------------------------------------------------
def trainer(device, **kw):
    cfg = GPTConfig(**{**CFG, "d_model": 256, "n_heads": 2, "ffn": 640, "vocab": 1000, "seq": 128, **kw})
    return Trainer(cfg, TrainConfig(global_batch=4, micro_batch=2, lr=1e-2, optimizer="muon", weight_decay=0.01), device=torch.device(device))


def batch(tr, step):
    return torch.randint(0, tr.cfg.vocab, (4, tr.cfg.seq + 1), generator=torch.Generator().manual_seed(step))


def test_steps_and_resume_cpu(tmp_path):
    small = dict(d_model=64, ffn=128, vocab=200, seq=12, gated="silu", head_rows=7)
    a = trainer("cpu", **small)
    losses = [a.train_step(batch(a, i)) for i in range(2)]
    save_checkpoint(str(tmp_path), 2, a.model, a.opt)
    losses.append(a.train_step(batch(a, 2)))
    assert all(math.isfinite(v) for v in losses)
    b = trainer("cpu", **small)
    load_checkpoint(str(tmp_path), 2, b.model, b.opt)
    assert b.train_step(batch(b, 2)) == losses[-1]
    assert torch.equal(a.p_sh, b.p_sh) and torch.equal(a.p_rep, b.p_rep)


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_block_against_its_layers(act):
    """One kernel for both projections against the two products and the elementwise kernels that a mesh of several devices runs."""
    tr = trainer("cuda", dtype=torch.bfloat16, gated=act)
    ff, n = tr.model.blocks[0].ff, 256
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, dy = (ShardedTensor(tr.mesh, {(0, 0): torch.randn(n, 256, device="cuda", generator=gen).bfloat16()}) for _ in range(2))
    y = ff.forward(x)
    dx = ff.backward(dy)
    grads = [l.grad.local().clone() for l in ff.layers()]
    for l in ff.layers():
        l.zero_grad()
    ff._whole = lambda x: False
    y2 = ff.forward(x)
    dx2 = ff.backward(dy)
    near = lambda a, b: (a.float() - b.float()).norm() <= 2.0 ** -6 * b.float().norm()      # some five roundings to bf16, half a step each
    assert near(y.local(), y2.local()) and near(dx.local(), dx2.local())
    assert all(near(a, l.grad.local()) for a, l in zip(grads, ff.layers()))


@gpu
def test_head_without_logits_against_the_one_with():
    a, b = (trainer("cuda", dtype=torch.bfloat16, gated="silu", head_rows=r) for r in (100, None))
    key = (0, 0)
    ids = batch(a, 0).cuda()
    tok, tgt = (ShardedTensor(a.mesh, {key: t.reshape(-1)}) for t in (ids[:, :-1], ids[:, 1:]))
    losses = [t.model.forward_backward(tok, tgt, tgt.local().numel()).local() for t in (a, b)]
    assert abs(losses[0] - losses[1]).item() < 2.0 ** -8 * losses[1].item()      # logits in 16 bits on one side
    near = lambda x, y: (x.float() - y.float()).norm() <= 2.0 ** -5 * y.float().norm()
    assert near(a.g_sh, b.g_sh) and near(a.g_rep, b.g_rep)
    scored = a.model.token_losses(tok, tgt).local()
    assert abs(scored.mean() - losses[0]).item() < 2.0 ** -16 * losses[0].item()


@gpu
def test_steps_gpu():
    """Steps of all of it; a second run has the same bits, and the update is the optimizer's alone."""
    runs = []
    for _ in range(2):
        tr = trainer("cuda", dtype=torch.bfloat16, gated="silu", head_rows=0)
        before = tr.opt.groups[0].master.clone()
        losses = [tr.train_step(batch(tr, i).pin_memory()) for i in range(3)]
        tr.check()
        assert all(math.isfinite(v) for v in losses)
        assert torch.isfinite(tr.opt.groups[0].master).all() and (tr.opt.groups[0].master - before).abs().max() > 0
        for w in tr.model.blocks[0].matrices():
            assert w.local().isfinite().all()
        runs.append((losses, tr))
    a, b = (r[1].model.blocks[1].ff.gate.weight.local() for r in runs)
    # embeddings' gradients are added in any order, so not bit by bit
    assert (a.float() - b.float()).norm() <= 2.0 ** -5 * b.float().norm()
