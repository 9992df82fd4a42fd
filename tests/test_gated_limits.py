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


# ----------------------------------------------------------------------------------------------
# gates of any size
# ----------------------------------------------------------------------------------------------
def tails64(x, act):
    """Activation and derivative with sigmoids that keep their small values; how far fp32 may be off, as a share of both: the exponent q has up to
    six roundings, and its product with log2 e two more, each of 2^-24 of q, which are shares of the exponential; exponential, division and the
    products beside it 16 more of 2^-24.  Below 2^-120 a sigmoid may be 0."""
    a, cubic = (1.0, 0.0) if act == "silu" else (2 * (2 / torch.pi) ** 0.5, 0.044715)
    q = a * (x + cubic * x ** 3)
    s, r = torch.sigmoid(q), torch.sigmoid(-q)
    share = (8 * q.abs().clamp_max(90) + 16) * 2.0 ** -24
    dq = a * (1 + 3 * cubic * x ** 2)
    bend = torch.where(s * r == 0, 0.0, x * dq * s * r)
    off = share * s + torch.where(s * r == 0, 0.0, (x * dq).abs() * (2 * share * s * r + 2.0 ** -22 * s)).abs()
    return x * s, s + bend, share * (x * s).abs() + 2.0 ** -120 * x.abs(), off + 2.0 ** -118 * (1 + x.abs())


def grid():
    fine = torch.linspace(-12, 12, 3073)
    far = torch.tensor([16., 40., 87., 89., 1e3, 1e6, 1e12, 1e13, 2e19, 1e20, 1e25, 1e30, 3e38])
    return torch.cat([fine, far, -far, torch.zeros(5)]).bfloat16()


@both
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_from_far_below_to_far_above(dev, act):
    x = grid()
    x = x[:x.numel() // 8 * 8]
    one = torch.ones_like(x)
    a, da, ea, eda = tails64(x.double(), act)
    h = F.gated_act(x.to(dev), one.to(dev), act)
    dg, du = F.gated_act_bwd(one.to(dev), x.to(dev), one.to(dev), act)
    for got, want, off in ((h, a, ea), (du, a, ea), (dg, da, eda)):
        got = got.double().cpu()
        bad = (got - want).abs() > off + base.BF * want.abs() + 2.0 ** -126
        assert not bad.any() and got.isfinite().all(), (x[bad], got[bad], want[bad])


@both
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_whose_activation_is_zero_beside_large_factors(dev, act):
    """The factors' product is beyond fp32, the gradients are not."""
    x = torch.tensor([-1e30, -1e20, -1e25, -1e30, -1e35, -3e38, -1e21, -1e30]).bfloat16().to(dev)
    big = torch.full_like(x, 1e19)
    dg, du = F.gated_act_bwd(big, x, big * 10, act)
    assert dg.count_nonzero() == 0 and du.count_nonzero() == 0


@both
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("tokens", [3, 24])
def test_a_block_with_far_gates(dev, act, tokens):
    """Gates of 1e4 and 2e19 and below -1e4 and -2e19: the activation is the gate or 0, its derivative 1 or 0."""
    x = torch.zeros(tokens, 8).bfloat16()
    size = torch.tensor([1e4, 1e-3, 2e19])[torch.arange(tokens) % 3]
    x[:, 0] = size * torch.where(torch.arange(tokens) // 3 % 2 == 0, 1, -1)
    wg, wu, wd = torch.zeros(8, 16).bfloat16(), torch.zeros(8, 16).bfloat16(), torch.eye(16).bfloat16()
    wg[0] = 1
    wu[0] = 2.0 ** -10
    dy = torch.ones(tokens, 16).bfloat16()
    args = [t.to(dev) for t in (x, wg, wu, wd)]
    y, saved = F.gated_ff_fwd(*args, act=act)
    alone = F.gated_ff_fwd(*args, act=act, keep=False)[0]
    dx, grads = F.gated_ff_bwd(dy.to(dev), *args, saved, act=act)
    g = x[:, :1].double()
    a, da, _, _ = tails64(g, act)
    h = a * g * 2.0 ** -10
    for got in (y, alone):
        assert (got.double().cpu() - h).abs().le(2.0 ** -7 * h.abs() + 1e-37).all()
    want = 16 * (g * 2.0 ** -10 * da + a * 2.0 ** -10)                     # 16 features of one kind each
    assert (dx[:, :1].double().cpu() - want).abs().le(2.0 ** -6 * (g.abs() * da.abs() + a.abs()) * 2.0 ** -6 + 1e-37).all() and dx[:, 1:].count_nonzero() == 0
    # the up weight's has x a, up to 4e38: beyond fp32 itself
    assert grads[0].isfinite().all() and grads[2].isfinite().all()


@gpu
@pytest.mark.parametrize("size,weight", [(1e-6, 1.0), (1e5, 1.0), (3e-20, 1e-6), (1e4, 1e4)])
def test_gpu_range_of_gelu(size, weight):
    base.run("cuda", base.data(140, 64, 72, 40, size=size, weight=weight), "gelu")


# ----------------------------------------------------------------------------------------------
# few tokens: ends of the units and parts that the contraction is taken in
# ----------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("layout,unit", [("nn", 32), ("nt", 128)])
@pytest.mark.parametrize("ctas", [1, 2, 4, 8])
@pytest.mark.parametrize("tokens", [5, 12])
def test_gpu_few_tokens_at_the_ends_of_units(layout, unit, ctas, tokens):
    """Eight warps of 1 to 8 CTAs take a unit each in turn: one unit less than a round, a round, 8 beyond, and beyond two rounds; as inputs of the gated
    product and as features of the plain one.  A warp's share is a few instructions, so sums are off as those of 512 products are, twice at most
    where a warp takes several rounds (an instruction is cut off at 2^-22 of the largest)."""
    once = 8 * ctas * unit
    for long in (once - unit, once, once + 8, 2 * once + unit - 8):
        for d, f, o in ((long, 16, 24), (24, long, 16)):
            args = base.data(tokens, d, f, o, seed=long)
            y, off = base.definition(*args, "silu")["y"]
            x, wg, wu, wd = (t.cuda() for t in (args[0], *(base.lay(w, layout) for w in args[1:4])))
            got = F.gated_ff_fwd(x, wg, wu, wd, up_layout=layout, down_layout=layout, keep=False)[0]
            base.near(got, (y, 2 * off))
