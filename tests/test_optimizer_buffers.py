"""What the optimizers' kernels take of a flat buffer, and what is refused before a step."""
import pytest
import torch

from meshslice_b200 import optim
from meshslice_b200.optim import AdamW, FlatGroup, Muon

gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
# types of parameters and gradients, first elements of both
BAD = [(F32, F32, 0, 0), (torch.float16, F32, 0, 0), (BF, torch.float16, 0, 0), (BF, torch.float64, 0, 0), (BF, F32, 2, 0), (BF, F32, 0, 1), (BF, BF, 0, 6)]
GOOD = [(BF, F32, 0, 0), (BF, BF, 0, 0), (BF, F32, 4, 8), (BF, BF, 12, 4)]


def buffers(device, types, first):
    return [torch.ones(256 + 16, dtype=t, device=device)[i:i + 256] for t, i in zip(types, first)]


@pytest.mark.parametrize("p,g,i,j", BAD)
def test_buffers_that_are_refused(p, g, i, j):
    with pytest.raises(ValueError):
        optim._check_buffers(*buffers("cpu", (p, g), (i, j)))
    with pytest.raises(ValueError):
        optim._check_buffers(torch.ones(64, 2, dtype=BF)[:, 0], torch.ones(64))


@pytest.mark.parametrize("p,g,i,j", GOOD)
def test_buffers_that_are_taken(p, g, i, j):
    optim._check_buffers(*buffers("cpu", (p, g), (i, j)))


@gpu
@pytest.mark.parametrize("kind", ["adamw", "muon"])
@pytest.mark.parametrize("p,g,i,j", BAD)
def test_gpu_refusals(kind, p, g, i, j):
    group = FlatGroup(*buffers("cuda", (p, g), (i, j)), "sharded")
    with pytest.raises(ValueError):
        AdamW([group]) if kind == "adamw" else Muon([group], [group.param[:64].view(8, 8)])


@gpu
@pytest.mark.parametrize("kind", ["adamw", "muon"])
@pytest.mark.parametrize("p,g,i,j", GOOD)
def test_gpu_steps_stay_in_their_buffers(kind, p, g, i, j):
    param, grad = (torch.ones(256 + 16, dtype=t, device="cuda") for t in (p, g))
    group = FlatGroup(param[i:i + 256], grad[j:j + 256], "sharded")
    opt = AdamW([group], lr=0.1) if kind == "adamw" else Muon([group], [group.param[:64].view(8, 8)], lr=0.1)
    opt.step()
    assert torch.equal(group.param, group.master.to(BF)) and (group.param < 1).all()
    assert (param[:i] == 1).all() and (param[i + 256:] == 1).all() and (grad == 1).all()
