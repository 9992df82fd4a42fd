"""Orthogonal update of matrices: CPU formulation and kernels against the polynomial in 64 bits."""
import pytest
import torch

from meshslice_b200.ops import functional as F
from meshslice_b200.ops.orthogonal import COEFFICIENTS

gpu = pytest.mark.gpu


def half(t, scale):
    """Rounded to fp16 beside ``scale``."""
    return (t * scale).half().double() / scale


def polynomial(g, steps=5, coefficients=COEFFICIENTS, rounded=False):
    """In 64 bits; ``rounded``: with the factors of the products rounded as the kernels round them."""
    a, b, c = coefficients
    r = half if rounded else (lambda t, s: t)
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    norm = x.square().sum((-2, -1), keepdim=True).sqrt()
    x = torch.where(norm == 0, 0.0, x / norm)
    for _ in range(steps):
        xs = r(x, 2.0 ** 10)
        q = r(xs @ xs.mT, 2.0 ** 10)
        x = a * x + r(b * q + c * (q @ q), 2.0 ** 8) @ xs
    return x.mT if tall else x


def matrices(kind, items, m, n, seed=0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)
    if kind == "noise":
        g = r(items, m, n)
    elif kind == "low rank":
        k = max(1, min(m, n) // 8)
        g = r(items, m, k) @ r(items, k, n) + 0.05 * r(items, m, n)
    else:                                      # singular values over four powers of ten
        k = min(m, n)
        u, v = torch.linalg.qr(r(items, m, k))[0], torch.linalg.qr(r(items, n, k))[0]
        g = u * torch.logspace(0, -4, k) @ v.mT
    return (g * 1e-3).to(dtype)


def check(got, g, **kw):
    """Twice the distance that the roundings of the factors alone make, and the rounding of the result."""
    want, model = polynomial(g.cpu(), **kw), polynomial(g.cpu(), rounded=True, **kw)
    bits = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -20
    off = (got.double().cpu() - want).flatten(-2).norm(dim=-1)
    allowed = 2 * (model - want).flatten(-2).norm(dim=-1) + bits * want.flatten(-2).norm(dim=-1)
    assert off.le(allowed).all(), (off / allowed)


SIZES = [(1, 1, 1), (1, 8, 8), (2, 1, 100), (3, 100, 1), (1, 64, 64), (2, 65, 63), (1, 130, 300), (2, 300, 130), (1, 257, 513), (3, 40, 1000),
         (2, 256, 256), (1, 255, 129), (1, 257, 256), (2, 20, 257), (2, 300, 1), (80, 33, 17)]


@pytest.mark.parametrize("size", SIZES[:8])
@pytest.mark.parametrize("kind", ["noise", "low rank"])
def test_cpu(size, kind):
    g = matrices(kind, *size)
    got = F.orthogonalize(g, out_dtype=torch.float32)
    want = polynomial(g)
    # fp32: a relative 2^-24 of X grows by the polynomial's slope at 0, 3.44 a step
    near = lambda a, b: (a.double() - b).norm() <= 2.0 ** -24 * 3.4445 ** 5 * 64 * b.norm() + 1e-12
    assert all(near(a, b) for a, b in zip(got, want))
    assert near(F.orthogonalize(g[0], out_dtype=torch.float32), want[0])       # products of a batch may sum in another order


def test_cpu_singular_values():
    s = torch.linalg.svdvals(F.orthogonalize(matrices("noise", 2, 60, 300)).float())
    assert s.min() > 0.6 and s.max() < 1.3


@gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["noise", "low rank", "falling"])
@pytest.mark.parametrize("size", SIZES)
def test_gpu(size, kind, dtype, out):
    g = matrices(kind, *size, dtype=dtype)
    check(F.orthogonalize(g.cuda(), out_dtype=out), g)


@gpu
@pytest.mark.parametrize("size", [(1, 1100, 700), (5, 512, 640), (1, 128, 4096), (40, 128, 128)])
def test_gpu_many_tiles(size):
    g = matrices("low rank", *size)
    check(F.orthogonalize(g.cuda()), g)


@gpu
@pytest.mark.parametrize("steps,coefficients", [(1, COEFFICIENTS), (2, (1.5, -0.5, 0.0)), (3, (1.875, -1.25, 0.375)), (12, COEFFICIENTS)])
def test_gpu_other_polynomials(steps, coefficients):
    for n in (180, 280):
        g = matrices("noise", 2, 100, n)
        check(F.orthogonalize(g.cuda(), steps=steps, coefficients=coefficients, out_dtype=torch.float32), g, steps=steps, coefficients=coefficients)


@gpu
@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e18, 1e30])
def test_gpu_range(size):
    """Squares of the values are beyond fp32."""
    for n in (130, 290):
        g = matrices("noise", 2, 70, n) * size
        check(F.orthogonalize(g.cuda()), g)


@gpu
@pytest.mark.parametrize("n", [130, 290])
def test_gpu_zeros_and_bad_values(n):
    g = matrices("noise", 4, 70, n)
    g[1] = 0
    g[2, 3, 5] = float("nan")
    got = F.orthogonalize(g.cuda())
    assert got[1].count_nonzero() == 0 and got[2].isnan().any()
    for i in (0, 3):
        check(got[i:i + 1], g[i:i + 1])


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("n", [130, 290])
def test_out_shares_memory_with_other_matrices(n, dev):
    """Results that lie where matrices that are still to be read are: as without that."""
    g = matrices("noise", 4, 70, n).to(dev)
    want = F.orthogonalize(g[:3], out_dtype=torch.float32)
    for first, to in ((0, 1), (1, 0)):
        t = torch.zeros(4, 70, n, device=dev)
        t[first:first + 3] = g[:3]
        F.orthogonalize(t[first:first + 3], out=t[to:to + 3])
        assert torch.equal(t[to:to + 3], want)
    square = matrices("noise", 2, 70, 70).to(dev)
    want = F.orthogonalize(square, out_dtype=torch.float32)
    F.orthogonalize(square, out=square.mT)
    assert torch.equal(square.mT, want)


@gpu
@pytest.mark.parametrize("n", [130, 290])
def test_gpu_layouts(n):
    """Strided batches, results in other layouts and in place; in one launch and in several."""
    g = matrices("noise", 3, 70, n)
    plain = F.orthogonalize(g.cuda())
    flat = torch.zeros(3, 70 * n + 28, device="cuda")
    view = flat.as_strided((3, 70, n), (70 * n + 28, n, 1))
    view.copy_(g)
    assert torch.equal(F.orthogonalize(view), plain)
    assert torch.equal(F.orthogonalize(g.mT.contiguous().mT.cuda()), plain)
    assert torch.equal(F.orthogonalize(g.mT.contiguous().cuda()).mT, plain)
    out = torch.zeros(3, 80, n + 10, dtype=torch.bfloat16, device="cuda")
    part = out[:, 5:75, 3:n + 3]
    assert F.orthogonalize(g.cuda(), out=part) is part and torch.equal(part, plain)
    part.zero_()
    assert out.count_nonzero() == 0
    out = torch.zeros(n, 70, 3, dtype=torch.bfloat16, device="cuda").permute(2, 1, 0)
    assert F.orthogonalize(g.cuda(), out=out) is out and torch.equal(out, plain)
    own = g.cuda()
    whole = F.orthogonalize(own, out_dtype=torch.float32)
    assert F.orthogonalize(own, out=own) is own and torch.equal(own, whole)


@gpu
def test_gpu_some_at_a_time(monkeypatch):
    """A batch that the workspace does not hold, on another stream; every matrix gets the same bits."""
    from meshslice_b200.ops import orthogonal
    g = matrices("noise", 5, 70, 290).cuda()
    plain = F.orthogonalize(g)
    monkeypatch.setattr(orthogonal, "WORKSPACE_BYTES", 900000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, plain)
    assert torch.equal(F.orthogonalize(g[2]), plain[2])


@gpu
@pytest.mark.parametrize("m", [130, 290])
def test_gpu_graphs(m):
    built = []
    for seed in (0, 1):
        g = matrices("noise", 2, m, 70, seed=seed).cuda()
        graph = torch.cuda.CUDAGraph()
        F.orthogonalize(g)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = F.orthogonalize(g)
        built.append((g, graph, out))
    for k, (g, _, _) in enumerate(built):
        g.copy_(matrices("noise", 2, m, 70, seed=5 + k))
    for _, graph, _ in built:
        graph.replay()
    torch.cuda.synchronize()
    for g, _, out in built:
        assert torch.equal(out, F.orthogonalize(g))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_empty(dev):
    assert F.orthogonalize(torch.zeros(0, 3, 4, device=dev)).shape == (0, 3, 4)
    assert F.orthogonalize(torch.zeros(3, 0, device=dev)).shape == (3, 0)


BAD = {
    "vector": lambda g: F.orthogonalize(g[0]),
    "type": lambda g: F.orthogonalize(g.double()),
    "no steps": lambda g: F.orthogonalize(g, steps=0),
    "half a step": lambda g: F.orthogonalize(g, steps=1.5),
    "two coefficients": lambda g: F.orthogonalize(g, coefficients=(1.5, -0.5)),
    "a polynomial that grows": lambda g: F.orthogonalize(g, coefficients=(6.0, 1.0, 1.0)),
    "one that is no number": lambda g: F.orthogonalize(g, coefficients=(1.5, float("nan"), 0.0)),
    "type of the result": lambda g: F.orthogonalize(g, out_dtype=torch.float16),
    "shape of the result": lambda g: F.orthogonalize(g, out=torch.zeros(4, 4, device=g.device)),
    "an out that lies on itself": lambda g: F.orthogonalize(g, out=torch.zeros(1, 6, device=g.device).expand(4, 6)),
    "a batch of one out": lambda g: F.orthogonalize(g.expand(3, 4, 6), out=torch.zeros(1, 4, 6, device=g.device).expand(3, 4, 6)),
    "type of out": lambda g: F.orthogonalize(g, out=torch.zeros(4, 6, device=g.device, dtype=torch.float64)),
}


@pytest.mark.parametrize("what", BAD)
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(dev, what):
    with pytest.raises(ValueError):
        BAD[what](torch.ones(4, 6, device=dev))
