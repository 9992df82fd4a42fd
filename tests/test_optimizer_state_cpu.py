"""Optimizer state between runs: what a moment means goes with it."""
import json

import pytest
import torch

from meshslice_b200.checkpoint import load_checkpoint, reshard_checkpoint, save_checkpoint
from meshslice_b200.models.gpt import GPTConfig
from meshslice_b200.optim import AdamW, FlatGroup, Muon
from meshslice_b200.trainer import Trainer, TrainConfig

CFG = dict(n_layers=1, d_model=32, n_heads=2, ffn=64, vocab=90, seq=8, vocab_pad=32, dtype=torch.float32, gated="silu")


def trainer(optimizer, **kw):
    return Trainer(GPTConfig(**{**CFG, **kw}), TrainConfig(global_batch=2, micro_batch=1, lr=1e-2, optimizer=optimizer), device=torch.device("cpu"))


def steps(tr, n):
    for i in range(n):
        tr.train_step(torch.randint(0, 90, (2, 9), generator=torch.Generator().manual_seed(i)))
    return tr


def forget(path):
    """The checkpoint as it was before it said what updated its parameters."""
    meta = json.loads(path.read_text())
    meta.pop("update_rules", None)
    path.write_text(json.dumps(meta))


@pytest.mark.parametrize("tagged", [True, False])
@pytest.mark.parametrize("a", ["adamw", "muon"])
@pytest.mark.parametrize("b", ["adamw", "muon"])
def test_checkpoint_of_the_same_and_of_another_optimizer(tmp_path, a, b, tagged):
    first, second = steps(trainer(a), 3), trainer(b, init_std=0.3)
    d = save_checkpoint(str(tmp_path), 3, first.model, first.opt)
    if not tagged:
        forget(tmp_path / "step_3" / "meta.json")
    before = second.p_sh.clone()
    if a == b:
        load_checkpoint(str(tmp_path), 3, second.model, second.opt)
        assert torch.equal(second.p_sh, first.p_sh) and second.opt.step_count == 3
        for x, y in zip(first.opt.groups, second.opt.groups):
            assert torch.equal(x.master, y.master) and torch.equal(x.m, y.m) and torch.equal(x.v, y.v)
        return
    with pytest.raises(ValueError, match="another optimizer"):
        load_checkpoint(str(tmp_path), 3, second.model, second.opt)
    assert torch.equal(second.p_sh, before) and second.opt.step_count == 0 and not second.opt.groups[0].m.any()
    load_checkpoint(str(tmp_path), 3, second.model)                      # the way on that the message names
    second.opt.resync_from_params(3)
    assert torch.equal(second.opt.groups[0].master, first.p_sh) and second.opt.step_count == 3
    assert d


@pytest.mark.parametrize("tagged", [True, False])
def test_resharded_checkpoint_keeps_its_rules(tmp_path, tagged):
    tr = steps(trainer("muon", gated=""), 2)
    save_checkpoint(str(tmp_path / "a"), 2, tr.model, tr.opt)
    if not tagged:
        forget(tmp_path / "a" / "step_2" / "meta.json")
    reshard_checkpoint(str(tmp_path / "a"), 2, (1, 2), str(tmp_path / "b"))
    reshard_checkpoint(str(tmp_path / "b"), 2, (1, 1), str(tmp_path / "c"))
    again = trainer("muon", gated="")
    load_checkpoint(str(tmp_path / "c"), 2, again.model, again.opt)
    assert torch.equal(again.opt.groups[0].m, tr.opt.groups[0].m)
    with pytest.raises(ValueError, match="another optimizer"):
        load_checkpoint(str(tmp_path / "c"), 2, *(lambda t: (t.model, t.opt))(trainer("adamw", gated="")))


@pytest.mark.parametrize("tagged", [True, False])
@pytest.mark.parametrize("a", ["adamw", "muon"])
@pytest.mark.parametrize("b", ["adamw", "muon"])
def test_state_dict_of_the_same_and_of_another_optimizer(a, b, tagged):
    def build(kind):
        gen = torch.Generator().manual_seed(0)
        group = FlatGroup(torch.randn(64 * 64 + 96, generator=gen), torch.randn(64 * 64 + 96, generator=gen), "sharded")
        return Muon([group], [group.param[64:64 + 64 * 64].view(64, 64)]) if kind == "muon" else AdamW([group])
    first, second = build(a), build(b)
    for _ in range(3):
        first.step()
    state = first.state_dict()
    if not tagged:
        for s in state["groups"]:
            s.pop("adamw", None)
    if a == b:
        second.load_state_dict(state)
        assert second.step_count == 3 and torch.equal(second.groups[0].m, first.groups[0].m)
        return
    with pytest.raises(ValueError, match="another optimizer"):
        second.load_state_dict(state)
    assert second.step_count == 0 and not second.groups[0].m.any()


def test_matrices_cut_otherwise_and_states_without_steps():
    """The rule counts, not how the elements are cut into matrices; a state that says nothing and holds nothing fits either."""
    def build(shape):
        group = FlatGroup(torch.ones(4096), torch.ones(4096), "sharded")
        n = 4096 // (shape[0] * shape[1])
        return Muon([group], [group.param[i * shape[0] * shape[1]:(i + 1) * shape[0] * shape[1]].view(shape) for i in range(n)])
    first, second = build((64, 64)), build((32, 64))
    first.step()
    second.load_state_dict(first.state_dict())
    assert torch.equal(second.groups[0].m, first.groups[0].m)
    state = build((64, 64)).state_dict()
    state["groups"][0].pop("adamw", None)
    AdamW([FlatGroup(torch.ones(4096), torch.ones(4096), "sharded")]).load_state_dict(state)
