"""Gated feed-forward block at the edges of what its documentation allows."""
import pytest
import torch

import test_gated as base
from meshslice_b200.ops import functional as F

gpu = pytest.mark.gpu
both = pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
D, FF, O = 24, 40, 32


def call(dev, build):
    """A backward pass that adds to what ``build(args)`` gives of the operands x, gate, up, down, dy."""
    args = [t.to(dev) for t in base.data(9, D, FF, O)]
    args, grads = build(args)
    x, wg, wu, wd, dy = args
    saved = F.gated_ff_fwd(x, wg, wu, wd)[1]
    return F.gated_ff_bwd(dy, x, wg, wu, wd, saved, grads=grads)[1], args


def zeros(args):
    return [torch.zeros_like(w) for w in args[1:4]]


def part(buf, at, rows, cols):
    return buf[at:at + rows * cols].view(rows, cols)


def two_that_overlap(a):
    buf = torch.zeros(2 * D * FF, dtype=a[1].dtype, device=a[1].device)
    return a, (part(buf, 0, D, FF), part(buf, 8, D, FF), torch.zeros_like(a[3]))


def rows_that_overlap(a):
    buf = torch.zeros(D + 1, FF, dtype=a[1].dtype, device=a[1].device)
    return a, (buf[:D], buf[1:], torch.zeros_like(a[3]))


def columns_that_overlap(a):
    buf = torch.zeros(D, 2 * FF, dtype=a[1].dtype, device=a[1].device)
    return a, (buf[:, :FF], buf[:, FF - 8:2 * FF - 8], torch.zeros_like(a[3]))


def one_within_another_type(a):
    buf = torch.zeros(D * FF, dtype=torch.float32, device=a[1].device)
    return a, (buf.view(D, FF), part(buf.view(torch.bfloat16), 8, D, FF), torch.zeros_like(a[3]))


def a_weight(a):
    g = zeros(a)
    g[1] = a[2]
    return a, g


def another_weight(a):
    g = zeros(a)
    g[0] = a[2]
    return a, g


def the_input(a):
    buf = torch.zeros(D * FF + 8, dtype=a[0].dtype, device=a[0].device)
    x = part(buf, D * FF + 8 - 9 * D, 9, D)
    x.copy_(a[0])
    return [x, *a[1:]], (part(buf, 0, D, FF), *zeros(a)[1:])


def the_gradient_above(a):
    buf = torch.zeros(FF * O, dtype=a[0].dtype, device=a[0].device)
    dy = part(buf, 0, 9, O)
    dy.copy_(a[4])
    return [*a[:4], dy], (*zeros(a)[:2], buf.view(FF, O))


@both
@pytest.mark.parametrize("build", [two_that_overlap, rows_that_overlap, columns_that_overlap, one_within_another_type, a_weight, another_weight, the_input,
                                   the_gradient_above], ids=lambda f: f.__name__)
def test_gradients_in_shared_memory_are_refused(dev, build):
    with pytest.raises(ValueError, match="memory"):
        call(dev, build)


@both
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_side_by_side_are_taken(dev, dtype):
    """Gate and up as columns, as rows, and as neighbours of one buffer, weights as columns of one matrix."""
    want, _ = call(dev, lambda a: (a, [w.to(dtype) for w in zeros(a)]))

    def columns(a):
        buf, w = torch.zeros(D, 2 * FF, dtype=dtype, device=dev), torch.cat(a[1:3], 1)
        return [a[0], w[:, :FF], w[:, FF:], *a[3:]], (buf[:, :FF], buf[:, FF:], torch.zeros(FF, O, dtype=dtype, device=dev))

    def neighbours(a):
        buf = torch.zeros(2 * D * FF + FF * O, dtype=dtype, device=dev)
        return a, (part(buf, 0, D, FF), part(buf, D * FF, D, FF), part(buf, 2 * D * FF, FF, O))
    for build in (columns, neighbours):
        got, _ = call(dev, build)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
