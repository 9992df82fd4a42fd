"""Gated feed-forward block: CPU formulation and kernels against its formula in 64 bits, element by element."""
import math

import pytest
import torch

from meshslice_b200.ops import functional as F

gpu = pytest.mark.gpu
BF, KEPT = 2.0 ** -8, 2.0 ** -11      # half a step of bf16, and of what is kept of gate and up
SUM = 2.0 ** -18                      # sums of up to 512 products of fp32, exponentials and divisions


def act64(g, act):
    """Activation, its derivative, a bound of its second derivative."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), 0.5
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g), 0.8


def definition(x, wg, wu, wd, dy, act):
    """Values and, from the roundings, how far each may be off: h, dg and du are rounded to bf16, gate and up kept with 11 bits (and those
    2^-28 below a chunk's largest with less), outputs rounded to bf16."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    g, u = x @ wg, x @ wu
    eg, eu = SUM * (x.abs() @ wg.abs()), SUM * (x.abs() @ wu.abs())
    a, da, dda = act64(g, act)
    h = a * u
    eh = 1.13 * eg * u.abs() + a.abs() * eu + (BF + SUM) * h.abs()
    y = h @ wd
    out = {"y": (y, eh @ wd.abs() + SUM * (h.abs() @ wd.abs()) + BF * y.abs())}
    dh = dy @ wd.T
    edh = SUM * (dy.abs() @ wd.abs().T)
    tiny = 2.0 ** -38
    kg, ku = eg + KEPT * g.abs() + tiny * g.abs().amax(1, keepdim=True), eu + KEPT * u.abs() + tiny * u.abs().amax(1, keepdim=True)
    dg, du = dh * u * da, dh * a
    edu = edh * a.abs() + dh.abs() * 1.13 * kg + (BF + SUM) * du.abs()
    edg = edh * (u * da).abs() + dh.abs() * (ku * (da.abs() + dda * kg) + u.abs() * (dda * kg + SUM)) + (BF + SUM) * dg.abs()
    dx = dg @ wg.T + du @ wu.T
    out["dx"] = (dx, edg @ wg.abs().T + edu @ wu.abs().T + 2 * SUM * (dg.abs() @ wg.abs().T + du.abs() @ wu.abs().T) + BF * dx.abs())
    for name, left, right, el, er in (("gate", x, dg, None, edg), ("up", x, du, None, edu), ("down", h, dy, eh, None)):
        v = left.T @ right
        e = 2 * SUM * (left.abs().T @ right.abs()) + (left.abs().T @ er if er is not None else el.T @ right.abs())
        out[name] = (v, e + BF * v.abs())
    return out


def data(n, d, f, o, seed=0, size=1.0, weight=1.0, dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)
    return [t.to(dtype) for t in (r(n, d) * size, r(d, f) * d ** -0.5 * weight, r(d, f) * d ** -0.5 * weight, r(f, o) * f ** -0.5, r(n, o))]


def lay(t, layout):
    return t if layout == "nn" else t.T.contiguous()


def near(got, want):
    value, off = want
    assert (got.double().cpu() - value).abs().le(off + 1e-37).all(), ((got.double().cpu() - value).abs() - off).max()


def run(dev, args, act="silu", up="nn", down="nn", grads=None, move=lambda t: t):
    x, wg, wu, wd, dy = args
    want = definition(x, wg, wu, wd, dy, act)
    x, wg, wu, wd, dy = (move(t.to(dev)) for t in (x, lay(wg, up), lay(wu, up), lay(wd, down), dy))
    y, saved = F.gated_ff_fwd(x, wg, wu, wd, act=act, up_layout=up, down_layout=down)
    alone, nothing = F.gated_ff_fwd(x, wg, wu, wd, act=act, up_layout=up, down_layout=down, keep=False)
    assert nothing is None
    if dev == "cpu" or x.shape[0] > 16:
        assert torch.equal(alone, y)
    else:                                # a kernel of its own, with the same roundings
        near(alone, want["y"])
    dx, dw = F.gated_ff_bwd(dy, x, wg, wu, wd, saved, act=act, up_layout=up, down_layout=down, grads=grads)
    near(y, want["y"])
    near(dx, want["dx"])
    if grads is None:
        for t, name, layout in zip(dw, ("gate", "up", "down"), (up, up, down)):
            assert t.dtype == x.dtype and t.is_contiguous()
            near(lay(t, layout) if layout == "nn" else t.T, want[name])
    return y, dx, dw, want


SIZES = [(1, 8, 8, 8), (3, 64, 40, 24), (130, 72, 200, 136), (300, 512, 264, 72), (257, 136, 1000, 128), (5, 24, 136, 264)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("size", SIZES[:3])
@pytest.mark.parametrize("up,down", [("nn", "nn"), ("nt", "nt")])
def test_cpu(size, act, up, down):
    run("cpu", data(*size), act, up, down)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_cpu_gradients_against_differences(act):
    args = [t.double() for t in data(3, 5, 7, 4, dtype=torch.float64)]
    x, wg, wu, wd, dy = args
    f = lambda *a: ((act64(a[0] @ a[1], act)[0] * (a[0] @ a[2])) @ a[3] * dy).sum()
    want = definition(x, wg, wu, wd, dy, act)
    for k, name in enumerate(("dx", "gate", "up", "down")):
        t = args[k]
        for i in range(0, t.numel(), 3):
            step = torch.zeros_like(t).view(-1)
            step[i] = 1e-5
            step = step.view_as(t)
            a, b = list(args[:4]), list(args[:4])
            a[k], b[k] = t + step, t - step
            assert abs((f(*a) - f(*b)).item() / 2e-5 - want[name][0].reshape(-1)[i].item()) < 1e-7


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("up,down", [("nn", "nn"), ("nt", "nt"), ("nn", "nt")])
@pytest.mark.parametrize("size", SIZES)
def test_gpu(size, act, up, down):
    run("cuda", data(*size), act, up, down)


@gpu
@pytest.mark.parametrize("up", ["nn", "nt"])
@pytest.mark.parametrize("down", ["nn", "nt"])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 16, 17])
def test_gpu_few_tokens(tokens, up, down):
    """Every number of tokens that has a kernel, and the one beyond; widths that end inside a CTA."""
    for d, f, o in ((8, 8, 8), (264, 72, 40), (512, 136, 24)):
        run("cuda", data(tokens, d, f, o, seed=tokens), "gelu" if tokens % 2 else "silu", up, down)


@gpu
@pytest.mark.parametrize("layout", ["nn", "nt"])
def test_gpu_few_tokens_long_contractions(layout):
    """Contractions of several pieces in shared memory: 4096 at a time."""
    gen = torch.Generator().manual_seed(0)
    d, f, o = 8200, 4104, 16
    x = torch.randn(5, d, generator=gen).bfloat16()
    wg, wu, wd = ((torch.randn(s, generator=gen) * s[0] ** -0.5).bfloat16() for s in ((d, f), (d, f), (f, o)))
    y, _ = F.gated_ff_fwd(x.cuda(), *(lay(w, layout).cuda() for w in (wg, wu, wd)), up_layout=layout, down_layout=layout, keep=False)
    near(y, [t * (8 if i else 1) for i, t in enumerate(definition(x, wg, wu, wd, torch.zeros(5, o), "silu")["y"])])     # longer sums


@gpu
def test_gpu_many_tiles():
    """More tiles than clusters, of every pass."""
    run("cuda", data(2100, 264, 1304, 256), "silu", "nn", "nt")


@gpu
@pytest.mark.parametrize("size,weight", [(1e-6, 1.0), (1e5, 1.0), (3e-20, 1e-6), (1e4, 1e4)])
def test_gpu_range(size, weight):
    """Projections far from 1: what is kept of them is not bound to the range of fp16."""
    run("cuda", data(140, 64, 72, 40, size=size, weight=weight))


@gpu
def test_gpu_strided_rows():
    """Rows that are part of wider ones, on and off a 16-byte boundary."""
    def wider(k):
        def move(t):
            w = torch.full((t.shape[0], t.shape[1] + 24), 7.0, dtype=t.dtype, device=t.device)
            w[:, k:k + t.shape[1]] = t
            return w[:, k:k + t.shape[1]]
        return move
    args = data(130, 72, 200, 136)
    plain = run("cuda", args)
    for k in (8, 3):
        got = run("cuda", args, move=wider(k))
        assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1]) and all(torch.equal(a, b) for a, b in zip(got[2], plain[2]))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_gradients_are_added(dtype):
    args = data(130, 72, 200, 136)
    shapes = (72, 200), (72, 200), (136, 200)
    base = [torch.randn(s, generator=torch.Generator().manual_seed(3)).to(dtype) for s in shapes]
    grads = tuple(t.clone().cuda() for t in base)
    _, _, dw, want = run("cuda", args, down="nt", grads=grads)
    assert all(a is b for a, b in zip(dw, grads))
    for t, b, name in zip(grads, base, ("gate", "up", "down")):
        value, off = want[name]
        value, off = (value.T, off.T) if name == "down" else (value, off)
        near(t, (value + b.double(), off + (BF if dtype == torch.bfloat16 else 2.0 ** -23) * (value + b.double()).abs()))


@gpu
def test_gpu_repeats_bit_by_bit_and_on_another_stream():
    args = [t.cuda() for t in data(300, 128, 264, 72)]
    x, wg, wu, wd, dy = args

    def both():
        y, saved = F.gated_ff_fwd(x, wg, wu, wd)
        return (y, *F.gated_ff_bwd(dy, x, wg, wu, wd, saved)[1])
    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@gpu
def test_gpu_graphs():
    """Two captured graphs with their own workspaces, replayed in turn on new inputs."""
    def build(seed):
        args = [t.cuda() for t in data(130, 72, 200, 136, seed=seed)]
        x, wg, wu, wd, dy = args

        def step():
            y, saved = F.gated_ff_fwd(x, wg, wu, wd)
            dx, dw = F.gated_ff_bwd(dy, x, wg, wu, wd, saved)
            return (y, dx, *dw)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return args, graph, out, step
    built = [build(s) for s in (0, 1)]
    for k, (args, _, _, _) in enumerate(built):
        for t, v in zip(args, data(130, 72, 200, 136, seed=10 + k)):
            t.copy_(v)
    for _, graph, _, _ in built:
        graph.replay()
    torch.cuda.synchronize()
    for _, _, out, step in built:
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


@gpu
def test_gpu_a_bad_token_stays_alone():
    x, wg, wu, wd, dy = (t.cuda() for t in data(300, 128, 264, 72))
    y, saved = F.gated_ff_fwd(x, wg, wu, wd)
    dx, _ = F.gated_ff_bwd(dy, x, wg, wu, wd, saved)
    bad = x.clone()
    bad[17] = float("nan")
    bad[200, 5] = float("inf")
    yb, saved = F.gated_ff_fwd(bad, wg, wu, wd)
    dxb, _ = F.gated_ff_bwd(dy, bad, wg, wu, wd, saved)
    others = torch.ones(300, dtype=torch.bool, device="cuda")
    others[[17, 200]] = False
    assert torch.equal(y[others], yb[others]) and torch.equal(dx[others], dxb[others])
    assert yb[17].isnan().all() and not yb[200].isfinite().all() and not dxb[200].isfinite().all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_no_tokens(dev):
    x, wg, wu, wd, dy = (t.to(dev) for t in data(0, 16, 24, 8))
    y, saved = F.gated_ff_fwd(x, wg, wu, wd)
    dx, dw = F.gated_ff_bwd(dy, x, wg, wu, wd, saved)
    assert y.shape == (0, 8) and dx.shape == (0, 16) and all(t.count_nonzero() == 0 for t in dw)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_product_by_itself(dev, act):
    gen = torch.Generator().manual_seed(0)
    g, u, dh = ((torch.randn(37, 24, generator=gen) * 3).bfloat16().to(dev) for _ in range(3))
    a, da, _ = act64(g.double().cpu(), act)
    h, (dg, du) = F.gated_act(g, u, act), F.gated_act_bwd(dh, g, u, act)
    for got, want in ((h, a * u.double().cpu()), (dg, dh.double().cpu() * u.double().cpu() * da), (du, dh.double().cpu() * a)):
        # what cancels in the derivative is of size 1: 2^-18 of the other factors
        near(got, (want, BF * want.abs() + SUM * (want.abs() + (dh.double() * u.double()).abs().cpu())))
    odd = torch.randn(24, 37, generator=gen).bfloat16().to(dev).T
    assert torch.equal(F.gated_act(odd, u, act), F.gated_act(odd.contiguous(), u, act))
    assert F.gated_act(g[:0], u[:0], act).shape == (0, 24)


BAD = {
    "activation": lambda a: F.gated_ff_fwd(*a[:4], act="relu"),
    "layout": lambda a: F.gated_ff_fwd(*a[:4], up_layout="tn"),
    "gate": lambda a: F.gated_ff_fwd(a[0], a[1][:, :8], *a[2:4]),
    "inputs": lambda a: F.gated_ff_fwd(a[0][:, :8], *a[1:4]),
    "down": lambda a: F.gated_ff_fwd(*a[:3], a[3][:8]),
    "type": lambda a: F.gated_ff_fwd(a[0], a[1], a[2].double(), a[3]),
    "three dimensions": lambda a: F.gated_ff_fwd(a[0][None], *a[1:4]),
    "dy": lambda a: F.gated_ff_bwd(a[4][:1], *a[:4], F.gated_ff_fwd(*a[:4])[1]),
    "nothing kept": lambda a: F.gated_ff_bwd(a[4], *a[:4], None),
    "kept by another call": lambda a: F.gated_ff_bwd(a[4], *a[:4], F.gated_ff_fwd(a[0][:2], *a[1:4])[1]),
    "gradients": lambda a: F.gated_ff_bwd(a[4], *a[:4], F.gated_ff_fwd(*a[:4])[1], grads=(torch.zeros(1), torch.zeros(1), torch.zeros(1))),
    "two gradients": lambda a: F.gated_ff_bwd(a[4], *a[:4], F.gated_ff_fwd(*a[:4])[1], grads=(torch.zeros_like(a[1]), torch.zeros_like(a[2]))),
    "one gradient twice": lambda a: F.gated_ff_bwd(a[4], *a[:4], F.gated_ff_fwd(*a[:4])[1], grads=[torch.zeros_like(a[1])] * 2 + [torch.zeros_like(a[3])]),
    "operands": lambda a: F.gated_act(a[0], a[4]),
    "operands' activation": lambda a: F.gated_act(a[0], a[0], "tanh"),
}


@pytest.mark.parametrize("what", BAD)
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(dev, what):
    with pytest.raises(ValueError):
        BAD[what]([t.to(dev) for t in data(3, 16, 24, 32)])


@gpu
def test_gpu_refusals():
    with pytest.raises(ValueError, match="multiples of 8"):
        F.gated_ff_fwd(*[t.cuda() for t in data(3, 16, 20, 32)[:4]])
    with pytest.raises(ValueError, match="bf16"):
        F.gated_ff_fwd(*[t.cuda() for t in data(3, 16, 24, 32, dtype=torch.float32)[:4]])
    with pytest.raises(ValueError):
        F.gated_ff_fwd(*[t.cuda() for t in data(3, 16, 24, 32)[:3]], data(3, 16, 24, 32)[3])
