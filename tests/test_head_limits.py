"""Loss of an output head at the edges of what its documentation allows."""
import pytest
import torch

import test_head_loss as base
from meshslice_b200.ops import functional as F

gpu = pytest.mark.gpu
both = pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
N, D, VOCAB, COLS = 300, 72, 203, 208


def the_weight(x, w, t):
    return x, w, t, w


def the_weight_shifted(x, w, t):
    buf = torch.zeros(D + 1, COLS, dtype=w.dtype, device=w.device)
    buf[:D] = w
    return x, buf[:D], t, buf[1:]


def the_input(x, w, t):
    buf = torch.zeros(N * D + D * COLS, dtype=x.dtype, device=x.device)
    mine = buf[:N * D].view(N, D)
    mine.copy_(x)
    return mine, w, t, buf[(N - 1) * D:(N - 1) * D + D * COLS].view(D, COLS)


def the_targets(x, w, t):
    buf = torch.zeros(D * COLS, dtype=torch.float32, device=x.device)
    mine = buf[128:128 + 2 * N].view(torch.int64)
    mine.copy_(t)
    return x, w, mine, buf.view(D, COLS)


@both
@pytest.mark.parametrize("rows", [0, 128])
@pytest.mark.parametrize("build", [the_weight, the_weight_shifted, the_input, the_targets], ids=lambda f: f.__name__)
def test_a_gradient_in_the_operands_memory_is_refused(dev, build, rows):
    x, w, t, dw = build(*(v.to(dev) for v in base.data(N, D, VOCAB, COLS)))
    with pytest.raises(ValueError, match="memory"):
        F.head_loss_grad(x, w, t, VOCAB, 0.25, dw=dw, rows=rows)


@both
def test_a_gradient_beside_the_weight_is_taken(dev):
    x, w, t = (v.to(dev) for v in base.data(N, D, VOCAB, COLS))
    want = F.head_loss_grad(x, w, t, VOCAB, 0.25, dw=torch.zeros_like(w))
    buf = torch.zeros(D, 2 * COLS, dtype=w.dtype, device=dev)
    buf[:, :COLS] = w
    got = F.head_loss_grad(x, buf[:, :COLS], t, VOCAB, 0.25, dw=buf[:, COLS:])
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(buf[:, :COLS], w)
