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


# ----------------------------------------------------------------------------------------------
# orthogonal updates: before the first step, not in the middle of it
# ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("kw", [dict(steps=0), dict(steps=1.5), dict(coefficients=(1.5, -0.5)), dict(coefficients=(1.5, float("nan"), 0.0)),
                                dict(coefficients=(6.0, 1.0, 1.0)), dict(steps=400, coefficients=(3.0, 0.0, 0.0))], ids=str)
def test_polynomials_are_refused_when_the_optimizer_is_made(dev, kw):
    group = FlatGroup(*buffers(dev, (BF, F32), (0, 0)), "sharded")
    with pytest.raises(ValueError):
        Muon([group], [group.param[:64].view(8, 8)], **kw)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_empty_matrices_are_refused(dev):
    group = FlatGroup(*buffers(dev, (BF, F32), (0, 0)), "sharded")
    for shape in ((0, 8), (8, 0)):
        with pytest.raises(ValueError):
            Muon([group], [group.param[:64].view(8, 8), group.param[64:64].view(shape)])


@gpu
def test_gpu_more_steps_than_the_kernels_take():
    group = FlatGroup(*buffers("cuda", (BF, F32), (0, 0)), "sharded")
    with pytest.raises(ValueError, match="steps"):
        Muon([group], [group.param[:64].view(8, 8)], steps=65, coefficients=(1.5, -0.5, 0.0))


def test_other_polynomials_are_taken():
    group = FlatGroup(*buffers("cpu", (F32, F32), (0, 0)), "sharded")
    Muon([group], [group.param[:64].view(8, 8)], steps=3, coefficients=[1.875, -1.25, 0.375]).step()
    assert group.param.isfinite().all()
