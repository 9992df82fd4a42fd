"""Attention within a window that keeps the first tokens: CPU formulation and kernels against dense attention in 64 bits."""
import math

import pytest
import torch

from meshslice_b200.ops import functional as F


def inputs(batch, seq, kv, group, D=128, seed=0, std=0.01):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(batch * seq, kv * (group + 2) * D, generator=g).bfloat16()
    return qkv, (torch.randn(batch * seq, kv * group * D, generator=g) * std).bfloat16()


def definition(qkv, dout, batch, seq, kv, group, window, sinks):
    """(out, lse, dqkv) in 64 bits; the gradient by autograd."""
    D = qkv.shape[1] // (kv * (group + 2))
    x = qkv.double().requires_grad_(True)
    t = x.view(batch, seq, kv, group + 2, D).permute(0, 2, 3, 1, 4)
    q, k, v = t[:, :, :group], t[:, :, group:group + 1], t[:, :, group + 1:]
    i, j = torch.arange(seq, device=x.device)[:, None], torch.arange(seq, device=x.device)[None, :]
    seen = (j <= i) & ((i - j < (window or seq)) | (j < sinks))
    s = (q @ k.transpose(-1, -2) / math.sqrt(D)).masked_fill(~seen, -math.inf)
    out = (torch.softmax(s, -1) @ v).permute(0, 3, 1, 2, 4).reshape(batch * seq, -1)
    out.backward(dout.double())
    return out.detach(), torch.logsumexp(s, -1).detach().view(batch, kv * group, seq), x.grad


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


# Roundings to bf16 are off by up to 2^-8 and by 2^-8 / sqrt(3) / sqrt(2) = 2^-9.3 in the mean square over a binade.  The output takes two
# (P, itself), the gradient of V two and all gradients together three, of random sign: 2^-9.3 times the root of 2 and 3, and half as much
# again for what is not random.
U = 2.0 ** -9.3
OUT, GRAD = 1.5 * 2 ** 0.5 * U, 1.5 * 3 ** 0.5 * U


def propagated(qkv, dout, batch, seq, kv, group, window, sinks):
    """What relative errors of 1 in every dS and in every element of the rounded output, of random sign, come to in dQ and dK (sums of
    squares).  An error d of the row sum of dO * O goes into every dS of its row as -P d scale: where a query sees few keys, or
    dP - delta is a small difference, that is more than the rounding of dS itself."""
    D, scale = 128, 1.0 / math.sqrt(128)
    t = qkv.double().view(batch, seq, kv, group + 2, D).permute(0, 2, 3, 1, 4)
    q, k, v = t[:, :, :group], t[:, :, group:group + 1], t[:, :, group + 1:]
    i, j = torch.arange(seq, device=t.device)[:, None], torch.arange(seq, device=t.device)[None, :]
    seen = (j <= i) & ((i - j < (window or seq)) | (j < sinks))
    p = torch.softmax((q @ k.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf), -1)
    do = dout.double().view(batch, seq, kv, group, D).permute(0, 2, 3, 1, 4)
    o = p @ v
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * scale
    row = (do * o).square().sum(-1, keepdim=True) * scale ** 2
    dq = (ds.square() * k.square().sum(-1).unsqueeze(-2)).sum() + (row * (p @ k).square()).sum()
    dk = ((ds.square() + p.square() * row) * q.square().sum(-1, keepdim=True)).sum()
    return dq, dk


SHAPES = [  # batch, seq, kv, group, window, sinks
    (1, 1, 1, 1, 0, 0), (2, 1, 1, 2, 4, 3), (1, 2, 1, 1, 1, 0), (3, 127, 2, 1, 64, 0), (2, 128, 1, 1, 128, 4), (2, 129, 1, 3, 1, 0),
    (1, 200, 2, 1, 64, 1), (2, 256, 2, 1, 0, 0), (1, 257, 1, 4, 129, 130), (1, 385, 2, 2, 127, 4), (1, 640, 1, 1, 200, 400),
    (2, 500, 3, 1, 128, 16), (1, 900, 1, 8, 300, 4), (1, 1000, 1, 2, 1, 1), (1, 777, 2, 1, 5000, 9), (1, 1153, 1, 1, 256, 128),
]


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] < 400])
def test_cpu(shape):
    batch, seq, kv, group, window, sinks = shape
    qkv, dout = inputs(batch, seq, kv, group, D=16)
    out, lse = F.window_attention_fwd(qkv, *shape)
    want, wl, wg = definition(qkv, dout, *shape)
    assert rel(out, want) < OUT and (lse.double() - wl).abs().max() < 1e-5
    assert rel(F.window_attention_bwd(dout, qkv, out, lse, *shape), wg) < GRAD


def test_gradient_against_differences():
    shape = (1, 9, 1, 2, 3, 2)
    qkv, dout = inputs(1, 9, 1, 2, D=4, std=1.0)
    qkv, dout = qkv.float(), dout.float()
    out, lse = F.window_attention_fwd(qkv, *shape)
    grad = F.window_attention_bwd(dout, qkv, out, lse, *shape)
    f = lambda t: (definition(t, dout, *shape)[0] * dout.double()).sum().item()
    for i in range(qkv.numel()):
        d = torch.zeros(qkv.numel(), dtype=torch.float64)
        d[i] = 1e-4
        d = d.view_as(qkv)
        assert abs((f(qkv.double() + d) - f(qkv.double() - d)) / 2e-4 - grad.view(-1)[i].item()) < 1e-5


def test_whole_window_is_causal_attention():
    qkv, _ = inputs(2, 40, 3, 1, D=16)
    a, b = F.window_attention_fwd(qkv, 2, 40, 3), F.attention_fwd(qkv, 2, 40, 3, causal=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def refusals(dev, D):
    qkv, dout = (t.to(dev) for t in inputs(2, 8, 1, 2, D))
    out, lse = F.window_attention_fwd(qkv, 2, 8, 1, 2, 4, 1)
    for args in ((2, 7, 1, 2), (2, 8, 3, 2), (2, 8, 0, 2), (2, 8, 1, 0), (2, 8, 1, 2, -1), (2, 8, 1, 2, 4, -1), (16, 0, 1, 2), (3, 8, 1, 2)):
        with pytest.raises(ValueError):
            F.window_attention_fwd(qkv, *args)
    a = (2, 8, 1, 2, 4, 1)
    for args in ((dout[:8], qkv, out, lse), (dout.float(), qkv, out, lse), (dout, qkv, out[:, :D], lse), (dout, qkv, out, lse[:1]),
                 (dout, qkv, out, lse.double())):
        with pytest.raises(ValueError):
            F.window_attention_bwd(*args, *a)


def test_refusals():
    refusals("cpu", 16)


# ---------------------------------------------------------------------------------------------- on a GPU
def on_gpu(shape, seed=0):
    from meshslice_b200 import _native
    batch, seq, kv, group, window, sinks = shape
    qkv, dout = (t.cuda() for t in inputs(batch, seq, kv, group, seed=seed))
    out, lse = F.window_attention_fwd(qkv, *shape)
    _native.check_status()
    dqkv = F.window_attention_bwd(dout, qkv, out, lse, *shape)
    _native.check_status()
    return qkv, dout, out, lse, dqkv


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES + [(4, 1200, 10, 1, 300, 4), (3, 2100, 4, 4, 700, 20), (40, 100, 5, 1, 30, 2), (1, 5000, 2, 3, 1024, 4)])
def test_kernel(shape):
    batch, seq, kv, group, window, sinks = shape
    qkv, dout, out, lse, dqkv = on_gpu(shape)
    want, wl, wg = definition(qkv, dout, *shape)
    assert rel(out, want) < OUT and (lse.double() - wl).abs().max() < 1e-5
    assert ((out.double() - want).abs() <= 2.0 ** -6 * want.abs().max()).all()
    # by parts: a fault in the smaller gradients would not show beside the largest
    part = lambda t: t.double().view(batch, seq, kv, group + 2, 128).split([group, 1, 1], 3)
    got, ref = part(dqkv), part(wg)
    assert rel(got[2], ref[2]) < GRAD
    for a, b, e in zip(got[:2], ref[:2], propagated(qkv, dout, *shape)):
        assert (a - b).norm() < 1.5 * U * (e + b.square().sum()).sqrt()
    for b in range(batch):
        for h in range(kv):
            assert rel(got[2][b, :, h], ref[2][b, :, h]) < 2 * GRAD


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 2000, 16, 1, 300, 4), (5, 1500, 16, 1, 200, 20), (3, 1700, 8, 3, 260, 16), (4, 1921, 16, 1, 0, 0),
                                   (2, 1800, 33, 1, 128, 9)])
def test_kernel_many_items(shape):
    """More than six query-major items an SM: the two kinds of gradient items in launches of their own."""
    test_kernel(shape)


@pytest.mark.gpu
def test_kernel_on_another_stream_and_in_a_graph():
    shape = (2, 333, 2, 2, 90, 4)
    qkv, dout, out, lse, dqkv = on_gpu(shape)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x, d = qkv.clone().mul_(1), dout.clone().mul_(1)
        o, l = F.window_attention_fwd(x, *shape)
        g = F.window_attention_bwd(d, x, o, l, *shape)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, out) and torch.equal(g, dqkv)
    x, d = torch.zeros_like(qkv), torch.zeros_like(dout)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, l = F.window_attention_fwd(x, *shape)
        g = F.window_attention_bwd(d, x, o, l, *shape)
    for times in (1, 2):
        x.copy_(qkv)
        d.copy_(dout)
        graph.replay()
        assert torch.equal(o, out) and torch.equal(l, lse) and torch.equal(g, dqkv)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 300, 2, 2, 100, 4), (3, 1100, 9, 2, 256, 4)])
def test_kernel_is_deterministic_and_reads_strided_tensors(shape):
    batch, seq, kv, group, window, sinks = shape
    qkv, dout, out, lse, dqkv = on_gpu(shape)
    again = F.window_attention_fwd(qkv, *shape)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    wide = lambda t, at: torch.zeros(t.shape[0], t.shape[1] + 24, dtype=t.dtype, device="cuda")[:, at:at + t.shape[1]].copy_(t)
    for at in (0, 8, 3):
        got = F.window_attention_fwd(wide(qkv, at), *shape)
        assert torch.equal(got[0], out) and torch.equal(got[1], lse)
        g = F.window_attention_bwd(wide(dout, at), wide(qkv, at), wide(out, at), lse.transpose(1, 2).contiguous().transpose(1, 2), *shape)
        assert torch.equal(g, dqkv)
    odd = torch.zeros(qkv.numel() + 1, dtype=qkv.dtype, device="cuda")[1:].view_as(qkv).copy_(qkv)
    assert torch.equal(F.window_attention_fwd(odd, *shape)[0], out)


@pytest.mark.gpu
def test_kernel_reads_nothing_beyond_its_sequence():
    """A sequence's results are the same whatever its neighbours hold, NaN included, and NaN shows in what sees it alone."""
    shape = (3, 201, 2, 2, 70, 3)
    qkv, dout, out, lse, dqkv = on_gpu(shape)
    bad = qkv.view(3, 201, -1).clone()
    bad[0], bad[2] = float("nan"), float("inf")
    dbad = dout.view(3, 201, -1).clone()
    dbad[0], dbad[2] = float("inf"), float("nan")
    o, l = F.window_attention_fwd(bad.view_as(qkv), *shape)
    g = F.window_attention_bwd(dbad.view_as(dout), bad.view_as(qkv), o, l, *shape)
    assert torch.equal(o[201:402], out[201:402]) and torch.equal(l[1], lse[1]) and torch.equal(g[201:402], dqkv[201:402])
    assert o[:201].isnan().all()


@pytest.mark.gpu
def test_kernel_large_scores():
    """Scores of several hundred: probabilities of one key, running maxima that grow by more than the lazy rescaling allows."""
    shape = (1, 700, 1, 2, 200, 4)
    qkv, dout = (t.cuda() for t in inputs(1, 700, 1, 2))
    qkv = (qkv.float() * 12).bfloat16()
    out, lse = F.window_attention_fwd(qkv, *shape)
    want, wl, _ = definition(qkv, dout, *shape)
    assert rel(out, want) < OUT and (lse.double() - wl).abs().max() < 2e-4
    qkv[:, :256] = -qkv[:, 256:384].repeat(1, 2)          # every query against its own key: the diagonal is the lowest score
    out, lse = F.window_attention_fwd(qkv, *shape)
    want, wl, _ = definition(qkv, dout, *shape)
    assert rel(out, want) < OUT and (lse.double() - wl).abs().max() < 2e-4


@pytest.mark.gpu
def test_kernel_matches_causal_attention_and_refusals():
    qkv, dout, out, lse, dqkv = on_gpu((2, 512, 3, 1, 0, 0))
    o, l = F.attention_fwd(qkv, 2, 512, 3, causal=True)
    assert rel(out, o.double()) < 2 * OUT and (l - lse).abs().max() < 1e-4
    assert rel(dqkv, F.attention_bwd(dout, qkv, o, l, 2, 512, 3, True).double()) < 2 * GRAD
    refusals("cuda", 128)
    with pytest.raises(ValueError):
        F.window_attention_fwd(qkv.float(), 2, 512, 3)
    with pytest.raises(ValueError):
        F.window_attention_fwd(qkv, 2, 512, 6)
    assert F.window_attention_fwd(qkv[:0], 0, 512, 3)[0].shape == (0, 384)


@pytest.mark.gpu
@pytest.mark.parametrize("sinks,dead", [(4, range(1, 301)), (4, range(4)), (40, range(39)), (0, range(1, 301))])
def test_kernel_keys_of_minus_infinity(sinks, dead):
    """Keys whose score is -inf have probability 0, where a query's first tiles have no others too; a query without any other is NaN."""
    shape = (1, 700, 1, 2, 200, sinks)
    qkv, _ = inputs(1, 700, 1, 2)
    x = qkv.view(700, 4, 128)
    x[:, :2, 0] = 1.0
    x[list(dead), 2, 0] = -math.inf
    out, _ = F.window_attention_fwd(qkv.cuda(), *shape)
    want, _, _ = definition(qkv, torch.zeros(700, 256), *shape)
    held = ~want.isnan().any(1)
    assert held.sum() >= 300 and (~held).any() == (0 in dead or sinks == 0)
    got = out.double().cpu()
    assert rel(got[held], want[held]) < OUT and got[~held].isnan().any(1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 300, 2, 2, 100, 0), (1, 700, 1, 1, 0, 0), (1, 640, 1, 2, 200, 4)])
def test_kernel_nan_in_the_scores_of_a_query(shape):
    """A NaN in a query is a NaN in every gradient of the keys and values that it sees, whichever unit made the exponential, and in its
    own; sequences and heads beside it stay as they are."""
    batch, seq, kv, group, window, sinks = shape
    qkv, dout, out, lse, dqkv = on_gpu(shape)
    dout = dout.masked_fill(dout == 0, 0.01)
    j = torch.arange(seq, device="cuda")
    for bad in list(range(seq - 40, seq)) + [0, 1, 130, 131, 147]:
        x = qkv.clone()
        x[bad, 3] = float("nan")                                # the first query head of the first key head
        o, l = F.window_attention_fwd(x, *shape)
        g = F.window_attention_bwd(dout, x, o, l, *shape).view(seq, kv, group + 2, 128)
        seen = (j <= bad) & ((bad - j < (window or seq)) | (j < sinks))
        assert g[seen, 0, group:].isnan().all() and g[bad, 0, 0].isnan().all() and l[0, 0, bad].isnan()
        if kv > 1:
            assert torch.equal(g[:, 1], F.window_attention_bwd(dout, qkv, out, lse, *shape).view_as(g)[:, 1])


def long_window(dev, D):
    qkv, dout = (t.to(dev) for t in inputs(1, 150, 1, 1, D))
    a = (1, 150, 1, 1)
    out, lse = F.window_attention_fwd(qkv, *a, 150, 0)
    grad = F.window_attention_bwd(dout, qkv, out, lse, *a, 150, 0)
    for window, sinks in ((1 << 31, 0), (1 << 70, 0), (1 << 32, 1 << 32), (1, 1 << 40)):
        o, l = F.window_attention_fwd(qkv, *a, window, sinks)
        assert torch.equal(o, out) and torch.equal(l, lse)
        assert torch.equal(F.window_attention_bwd(dout, qkv, o, l, *a, window, sinks), grad)


def test_window_beyond_32_bits():
    """A window or a number of first tokens beyond the sequence is the whole sequence, however large."""
    long_window("cpu", 16)


@pytest.mark.gpu
def test_kernel_window_beyond_32_bits():
    long_window("cuda", 128)


def check_gradient(shape, qkv, dout, dqkv, wg):
    batch, seq, kv, group, window, sinks = shape
    part = lambda t: t.double().view(batch, seq, kv, group + 2, 128).split([group, 1, 1], 3)
    got, ref = part(dqkv), part(wg)
    assert rel(got[2], ref[2]) < GRAD
    for a, b, e in zip(got[:2], ref[:2], propagated(qkv, dout, *shape)):
        assert (a - b).norm() < 1.5 * U * (e + b.square().sum()).sqrt()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 700, 1, 2, 200, 4), (2, 500, 2, 1, 0, 0), (1, 900, 1, 2, 130, 20)])
def test_kernel_gradient_of_large_scores(shape):
    """Scores of several hundred: most probabilities are 0 or 1.  A score is off by some 2^-22 of the sum of its terms' sizes, of about a
    thousand: 2^-12 of a probability, beside 2^-9.3 for its rounding."""
    batch, seq, kv, group, window, sinks = shape
    qkv, dout = (t.cuda() for t in inputs(batch, seq, kv, group))
    qkv = (qkv.float() * 12).bfloat16()
    for _ in range(2):
        out, lse = F.window_attention_fwd(qkv, *shape)
        _, _, wg = definition(qkv, dout, *shape)
        check_gradient(shape, qkv, dout, F.window_attention_bwd(dout, qkv, out, lse, *shape), wg)
        x = qkv.view(batch * seq, kv, group + 2, 128)           # then every query against its own key: the diagonal is the lowest score
        x[:, :, :group] = -x[:, :, group:group + 1]


@pytest.mark.gpu
@pytest.mark.parametrize("sinks,dead", [(4, range(1, 301)), (40, range(1, 39)), (40, range(1, 301)), (1, range(300, 420))])
def test_kernel_gradient_of_keys_of_minus_infinity(sinks, dead):
    """Keys whose score is -inf for every query get no gradient and disturb nobody else's; only the queries' feature that meets the
    infinity is NaN, by the definition too."""
    shape = (1, 700, 1, 2, 200, sinks)
    qkv, dout = (t.cuda() for t in inputs(1, 700, 1, 2))
    x = qkv.view(700, 4, 128)
    x[:, :2, 0] = 1.0
    x[list(dead), 2, 0] = -math.inf
    out, lse = F.window_attention_fwd(qkv, *shape)
    g = F.window_attention_bwd(dout, qkv, out, lse, *shape).double().view(700, 4, 128)
    want = definition(qkv, dout, *shape)[2].view(700, 4, 128)
    assert g[:, 2:].isfinite().all() and want[:, 2:].isfinite().all() and g[:, :2, 1:].isfinite().all()
    assert (g[list(dead), 2:].abs() < 2.0 ** -100).all()
    # (the errors that go into dQ and dK, with the dead keys' infinity out of the sums: they have no probability)
    y = qkv.clone()
    y.view(700, 4, 128)[list(dead), 2, 0] = -20000.0
    assert rel(g[:, 3], want[:, 3]) < GRAD
    dq, dk = propagated(y, dout, *shape)
    for a, b, e in ((g[:, :2, 1:], want[:, :2, 1:], dq), (g[:, 2], want[:, 2], dk)):
        assert (a - b).norm() < 1.5 * U * (e + b.square().sum()).sqrt()
