"""Loss of an output head without its logits in memory: CPU formulation and kernels against its formula in 64 bits, element by element."""
import math

import pytest
import torch

from meshslice_b200.ops import functional as F

gpu = pytest.mark.gpu
BF = 2.0 ** -8
SUM = 2.0 ** -18      # sums of up to 512 products of fp32


def definition(x, w, targets, vocab, scale):
    """(loss, dx, dw) with how far each may be off: logits are sums in fp32, probabilities come from exponentials with 11 bits (or 2^-25 of the
    row's largest) and are rounded to bf16, gradients too."""
    x, w = x.double(), w.double()[:, :vocab]
    z = x @ w
    ez = SUM * (x.abs() @ w.abs()) + 2.0 ** -22 * (z - z.amax(1, keepdim=True)).abs().clamp_max(200)
    label = (targets >= 0) & (targets < vocab)
    y = torch.where(label, targets, 0)[:, None]
    logp = torch.log_softmax(z, 1)
    loss = torch.where(label, -logp.gather(1, y)[:, 0], 0.0)
    eloss = torch.where(label, 2 * ez.amax(1) + 2.0 ** -20 * (1 + torch.logsumexp(z, 1).abs() + z.gather(1, y)[:, 0].abs()), 0.0)
    p = logp.exp() * label[:, None] * scale
    ep = p * (2.0 ** -11 + 2.0 ** -19 + 2 * ez.amax(1, keepdim=True)) + 2.0 ** -24 * p.amax(1, keepdim=True)
    dz = p.clone()
    dz.scatter_add_(1, y, -scale * label[:, None].double())
    edz = ep + BF * dz.abs()
    dx, dw = dz @ w.T, x.T @ dz
    return ((loss, eloss), (dx, edz @ w.abs().T + 2 * SUM * (dz.abs() @ w.abs().T) + BF * dx.abs()),
            (dw, x.abs().T @ edz + 2 * SUM * (x.abs().T @ dz.abs()) + BF * dw.abs()))


def data(n, d, vocab, cols, missing=False, seed=0, std=2.0):
    gen = torch.Generator().manual_seed(seed)
    x, w = torch.randn(n, d, generator=gen).bfloat16(), (torch.randn(d, cols, generator=gen) * std * d ** -0.5).bfloat16()
    targets = torch.randint(0, vocab, (n,), generator=gen)
    if missing:
        targets[1::3] = -1
        targets[2::5] = vocab
    else:
        targets[-1] = vocab - 1
    return x, w, targets


def near(got, want):
    value, off = want
    assert (got.double().cpu() - value).abs().le(off + 1e-37).all(), ((got.double().cpu() - value).abs() - off).max()


def run(dev, x, w, targets, vocab, layout="nn", rows=0, scale=0.25):
    want = definition(x, w, targets, vocab, scale)
    wl = w if layout == "nn" else w.T.contiguous()
    x, wl, t = x.to(dev), wl.to(dev), targets.to(dev)
    loss, dx, dw = F.head_loss_grad(x, wl, t, vocab, scale, layout=layout, rows=rows)
    assert loss.dtype == torch.float32 and dx.dtype == x.dtype and dw.dtype == w.dtype and dw.shape == wl.shape
    near(loss, want[0])
    near(F.head_loss(x, wl, t, vocab, layout=layout), want[0])
    near(dx, want[1])
    dw = dw if layout == "nn" else dw.T
    near(dw[:, :vocab], want[2])
    assert dw[:, vocab:].count_nonzero() == 0
    return loss, dx, dw


# tokens, inputs, vocabulary, columns
SIZES = [(1, 8, 1, 8), (3, 64, 40, 40), (130, 72, 203, 208), (7, 512, 1000, 1152), (300, 136, 500, 512), (257, 24, 2111, 2112)]


@pytest.mark.parametrize("missing", [False, True])
@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("size", SIZES[:4])
def test_cpu(size, layout, missing):
    run("cpu", *data(*size, missing=missing), size[2], layout)


def test_cpu_gradients_against_differences():
    x, w, t = data(4, 5, 7, 8, missing=True)
    x, w = x.double(), w.double()
    f = lambda x, w: definition(x, w, t, 7, 0.25)[0][0].sum() * 0.25
    _, (dx, _), (dw, _) = definition(x, w, t, 7, 0.25)
    for i in range(x.numel()):
        step = torch.zeros(x.numel(), dtype=torch.float64)
        step[i] = 1e-5
        assert abs((f(x + step.view_as(x), w) - f(x - step.view_as(x), w)).item() / 2e-5 - dx.reshape(-1)[i].item()) < 1e-8
    for i in range(5):
        for j in range(7):
            step = torch.zeros_like(w)
            step[i, j] = 1e-5
            assert abs((f(x, w + step) - f(x, w - step)).item() / 2e-5 - dw[i, j].item()) < 1e-8


@gpu
@pytest.mark.parametrize("missing", [False, True])
@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("size", SIZES)
def test_gpu(size, layout, missing):
    run("cuda", *data(*size, missing=missing), size[2], layout)


@gpu
@pytest.mark.parametrize("layout", ["nn", "nt"])
def test_gpu_odd_vocabularies(layout):
    """Every width of the last tile, with padding behind it or (as a table) without."""
    for vocab in (5, 63, 64, 65, 127, 129, 255, 256, 257, 321):
        run("cuda", *data(9, 24, vocab, -(-vocab // 8) * 8 if layout == "nn" else vocab), vocab, layout)


@gpu
@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("n,d,vocab,rows", [(1, 24, 9001, 0), (33, 136, 12000, 0), (300, 72, 8200, 0), (100, 72, 8200, 33), (40, 520, 5000, 0)])
def test_gpu_few_tokens_large_vocabularies(n, d, vocab, rows, layout):
    """The contraction over the vocabulary in parts, the last of them shorter; with pieces of the tokens, the last of which has fewer."""
    run("cuda", *data(n, d, vocab, -(-vocab // 8) * 8, missing=n > 10), vocab, layout, rows)


@gpu
@pytest.mark.parametrize("d", [1024, 1032, 2056, 4096])
def test_gpu_contractions_in_parts(d):
    """Inputs beyond 1024 are summed in several accumulators: a loss is as near as sums in fp32 are, whatever the width."""
    x, w, t = data(70, d, 300, 320)
    w[:, t[:35]] += (x[:35].float() * 0.1).bfloat16().T                   # confident ones, whose logits are large
    z = x.double() @ w.double()[:, :300]
    want = -torch.log_softmax(z, 1).gather(1, t[:, None])[:, 0]
    loss = F.head_loss(x.cuda(), w.cuda(), t.cuda(), 300)
    # 64 sums of 16 products, each cut off by at most 2^-23 of the largest partial sum, and those of the parts: 2^-16 of |x| |w| at the very most,
    # 2^-21 of the logits in the mean (a quarter of 64 half steps, logits of few units)
    assert (loss.double().cpu() - want).norm() <= 2.0 ** -20 * (want.norm() + z.amax(1).norm())


@gpu
def test_gpu_many_tiles():
    run("cuda", *data(2100, 64, 5003, 5120), 5003)


@gpu
@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("rows", [1, 100, 256, 300, 10000])
def test_gpu_in_pieces(layout, rows):
    """Some rows at a time, with a last piece that is shorter: sums of the weight's gradient are held in fp32."""
    n = 5 if rows == 1 else 300
    run("cuda", *data(n, 72, 203, 320, missing=True), 203, layout, rows)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("rows", [0, 128])
def test_gpu_gradient_is_added(dtype, layout, rows):
    x, w, t = data(300, 72, 203, 320)
    want = definition(x, w, t, 203, 0.25)[2]
    base = torch.randn(72, 320, generator=torch.Generator().manual_seed(1)).to(dtype)
    dw = (base if layout == "nn" else base.T.contiguous()).cuda()
    got = F.head_loss_grad(x.cuda(), (w if layout == "nn" else w.T.contiguous()).cuda(), t.cuda(), 203, 0.25, layout=layout, dw=dw, rows=rows)[2]
    assert got is dw
    dw = dw.cpu() if layout == "nn" else dw.cpu().T
    assert torch.equal(dw[:, 203:], base[:, 203:])
    total = want[0] + base[:, :203].double()
    near(dw[:, :203], (total, want[1] + (BF if dtype == torch.bfloat16 else 2.0 ** -22) * (total.abs() + base[:, :203].double().abs())))


@gpu
def test_gpu_padding_does_not_matter():
    """Columns behind the vocabulary may hold anything."""
    for layout in ("nn", "nt"):
        x, w, t = data(130, 72, 203, 320)
        clean = run("cuda", x, w, t, 203, layout)
        w[:, 203:] = float("nan")
        w[:, 210:] = float("inf")
        again = F.head_loss_grad(x.cuda(), (w if layout == "nn" else w.T.contiguous()).cuda(), t.cuda(), 203, 0.25, layout=layout)
        assert torch.equal(again[0], clean[0]) and torch.equal(again[1], clean[1])
        dw = again[2] if layout == "nn" else again[2].T
        assert torch.equal(dw, clean[2])


@gpu
def test_gpu_hidden_columns():
    """Columns whose logits are -inf or the type's lowest value, a whole tile of them too, have no probability."""
    for low in (-math.inf, torch.finfo(torch.bfloat16).min):
        x, w, t = data(40, 16, 700, 704)
        x = x.abs() + 0.1
        w[:, 100:] = 0
        w[:, 130:] = low
        x[:, 1:] = 0                       # logits are x[:, 0] w[0]
        w[0, :130] = torch.linspace(-2, 2, 130).bfloat16()
        t = t % 130
        z = (x.double()[:, :1] * w.double()[0, :700])
        want = -torch.log_softmax(z, 1).gather(1, t[:, None])[:, 0]
        # the columns are named row by row, since zeros times -inf are no numbers
        w2 = w.clone()
        w2[1:] = 0
        loss, _, dw = F.head_loss_grad(x.cuda(), w2.cuda(), t.cuda(), 700, 1.0)
        if low == -math.inf:
            assert loss.isnan().logical_not().all()
        assert (loss.double().cpu() - want).abs().max() < 2.0 ** -18 * 20
        assert dw[:, 130:].count_nonzero() == 0


@gpu
def test_gpu_a_bad_token_stays_alone():
    x, w, t = (v.cuda() for v in data(300, 72, 203, 208))
    loss, dx, _ = F.head_loss_grad(x, w, t, 203, 1.0)
    bad = x.clone()
    bad[17, 3] = float("nan")
    bad[200, 3] = float("inf")
    bl, bdx, _ = F.head_loss_grad(bad, w, t, 203, 1.0)
    others = torch.ones(300, dtype=torch.bool, device="cuda")
    others[[17, 200]] = False
    assert torch.equal(loss[others], bl[others]) and torch.equal(dx[others], bdx[others])
    assert bl[[17, 200]].isnan().all()
    t[17] = -1                      # without a label nothing of it is left
    bl, bdx, dw = F.head_loss_grad(bad[:100], w, t[:100], 203, 1.0)
    assert bl[17] == 0 and bdx[17].count_nonzero() == 0
    assert torch.equal(bl[others[:100]], loss[:100][others[:100]])


@gpu
def test_gpu_strides_streams_and_graphs():
    x, w, t = (v.cuda() for v in data(130, 72, 203, 208))
    plain = F.head_loss_grad(x, w, t, 203, 1.0)
    wide = torch.full((130, 99), 3.0, dtype=x.dtype, device="cuda")
    wide[:, 5:77] = x
    tt = torch.stack([t, t], 1)[:, 0]
    got = F.head_loss_grad(wide[:, 5:77], w.T.contiguous().T, tt, 203, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(plain, got))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.head_loss_grad(x, w, t, 203, 1.0, rows=128)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    graphs = []
    for seed in (3, 4):
        args = [v.cuda() for v in data(130, 72, 203, 208, seed=seed)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = F.head_loss_grad(*args, 203, 1.0, rows=128)
        graphs.append((args, graph, out))
    for k, (args, _, _) in enumerate(graphs):
        for a, b in zip(args, data(130, 72, 203, 208, seed=20 + k)):
            a.copy_(b)
    for _, graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for args, _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, F.head_loss_grad(*args, 203, 1.0, rows=128)))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_no_tokens_no_labels(dev):
    x, w, t = (v.to(dev) for v in data(6, 16, 40, 64))
    loss, dx, dw = F.head_loss_grad(x[:0], w, t[:0], 40, 1.0)
    assert loss.shape == (0,) and dx.shape == (0, 16) and dw.shape == w.shape and dw.count_nonzero() == 0
    assert F.head_loss(x[:0], w, t[:0], 40).shape == (0,)
    loss, dx, dw = F.head_loss_grad(x, w, torch.full_like(t, -1), 40, 1.0)
    assert loss.count_nonzero() == 0 and dx.count_nonzero() == 0 and dw.count_nonzero() == 0


BAD = {
    "layout": lambda x, w, t: F.head_loss(x, w, t, 40, layout="tn"),
    "inputs": lambda x, w, t: F.head_loss(x[:, :8], w, t, 40),
    "vocabulary": lambda x, w, t: F.head_loss(x, w, t, 65),
    "no vocabulary": lambda x, w, t: F.head_loss(x, w, t, 0),
    "targets": lambda x, w, t: F.head_loss(x, w, t[:2], 40),
    "type of targets": lambda x, w, t: F.head_loss(x, w, t.int(), 40),
    "type": lambda x, w, t: F.head_loss(x, w.double(), t, 40),
    "dw": lambda x, w, t: F.head_loss_grad(x, w, t, 40, 1.0, dw=torch.zeros_like(w)[:, :8]),
    "type of dw": lambda x, w, t: F.head_loss_grad(x, w, t, 40, 1.0, dw=torch.zeros_like(w, dtype=torch.float64)),
    "rows": lambda x, w, t: F.head_loss_grad(x, w, t, 40, 1.0, rows=-1),
    "vector": lambda x, w, t: F.head_loss(x[0], w, t, 40),
}


@pytest.mark.parametrize("what", BAD)
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(dev, what):
    with pytest.raises(ValueError):
        BAD[what](*(v.to(dev) for v in data(6, 16, 40, 64)))


@gpu
def test_gpu_refusals():
    x, w, t = (v.cuda() for v in data(6, 16, 40, 64))
    for bad in (lambda: F.head_loss(x.float(), w.float(), t, 40), lambda: F.head_loss(x[:, :12], w[:12], t, 40),
                lambda: F.head_loss(x, w[:, :60].contiguous(), t, 40), lambda: F.head_loss(x, w, t.cpu(), 40),
                lambda: F.head_loss(x, w.cpu(), t, 40)):
        with pytest.raises(ValueError):
            bad()
