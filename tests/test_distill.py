"""Distillation loss and gradient: CPU formulation and kernels against the definition in 64 bits."""
import math

import pytest
import torch

from meshslice_b200.ops import functional as F
from meshslice_b200.ops.distill import distill_rescale


def definition(z, ids, values, targets, vocab, T, w):
    """(loss, d loss / d z, sum of the absolute parts of the loss, of the gradient) in 64 bits, row by row.  Not for NaN."""
    n, cols = z.shape
    loss, grad = torch.zeros(n, dtype=torch.float64), torch.zeros(n, cols, dtype=torch.float64)
    size, parts = torch.ones(n, dtype=torch.float64), torch.zeros(n, cols, dtype=torch.float64)
    for r in range(n):
        x = z[r, :vocab].double()
        kept = [(int(i), float(v)) for i, v in zip(ids[r], values[r]) if 0 <= int(i) < vocab and float(v) != -math.inf]
        if kept and w != 1.0:
            e = torch.softmax(torch.tensor([v for _, v in kept], dtype=torch.float64) / T, 0)
            p = torch.zeros(vocab, dtype=torch.float64)
            for (i, _), q in zip(kept, e):
                p[i] += q
            logq = torch.log_softmax(x / T, 0)
            # entries of one id are one event each with that token's probability under the student
            terms = [q * (q.log() - logq[i]) for (i, _), q in zip(kept, e) if q > 0]
            loss[r] += (1 - w) * T * T * sum(terms)
            size[r] += T * T * (1 + (e * e.clamp_min(1e-300).log()).sum().abs() + torch.logsumexp(x / T, 0).abs() + x.max().abs()) \
                + T * (p * torch.where(p > 0, (x - x.max()).abs(), 0.0)).sum()
            grad[r, :vocab] += (1 - w) * T * (logq.exp() - p)
            parts[r, :vocab] += (1 - w) * T * (logq.exp() + p)
        y = -1 if targets is None else int(targets[r])
        if 0 <= y < vocab and w != 0.0:
            logq = torch.log_softmax(x, 0)
            loss[r] -= w * logq[y]
            size[r] += torch.logsumexp(x, 0).abs() + (x[y] - x.max()).abs() + x.max().abs()
            hot = torch.zeros(vocab, dtype=torch.float64)
            hot[y] = 1
            grad[r, :vocab] += w * (logq.exp() - hot)
            parts[r, :vocab] += w * (logq.exp() + hot)
    return loss, grad, size, parts


def data(rows, vocab, cols, top, missing=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, cols, generator=g) * 2).bfloat16()
    ids = torch.stack([torch.randperm(vocab, generator=g)[:top] for _ in range(rows)]) if top else torch.zeros(rows, 0, dtype=torch.int64)
    values = torch.randn(rows, top, generator=g) * 3
    targets = torch.randint(0, vocab, (rows,), generator=g)
    if missing:
        ids[0::3, top // 2:] = -1
        ids[1::4] = vocab
        values[2::5, : top // 2 + 1] = -math.inf
        targets[1::3] = -1
    elif top:
        targets[::2] = ids[::2, 0]                     # labels among the entries
    return z, ids, values, targets


def check(got, want, scale, bits=20):
    """Loss: exponentials are 2^-22 off, sums and logarithms 2^-23 a step: 2^-19 of the absolute parts.  Gradient: half a unit of
    bf16 (2^-8), and of its parts 2^-17: the exponent (z - m) / T, up to 2^5, is rounded to 24 bits."""
    loss, grad = got
    wl, wg, size, parts = want
    assert ((loss.double().cpu() - wl).abs() <= 2.0 ** -19 * size).all()
    bound = 2.0 ** -8 * wg.abs() * scale + 2.0 ** -17 * parts * scale + 1e-37
    assert ((grad.double().cpu() - wg * scale).abs() <= bound).all()


SETTINGS = [(1.0, 0.0), (1.0, 0.3), (2.0, 0.0), (2.0, 0.5), (0.7, 1.0), (4.0, 0.1)]
SIZES = [(1, 1, 8, 1), (5, 203, 208, 9), (17, 1000, 1024, 33), (3, 9, 16, 9), (2, 40, 40, 0)]


def run(dev, size, T, w, missing, values_dtype=torch.float32, use_targets=True, in_place=False):
    rows, vocab, cols, top = size
    z, ids, values, targets = data(rows, vocab, cols, top, missing)
    values = values.to(values_dtype)
    t = targets if use_targets else None
    want = definition(z, ids, values, t, vocab, T, w)
    a = [x.to(dev) if x is not None else None for x in (z, ids, values, t)]
    got = F.distill_loss_grad(a[0], a[1], a[2], vocab, 0.25, temperature=T, targets=a[3], hard_weight=w, out=a[0] if in_place else None)
    check(got, want, 0.25)
    assert got[1][:, vocab:].count_nonzero() == 0
    if in_place:
        assert got[1] is a[0]
    else:
        assert torch.equal(a[0].cpu(), z)
    return got


@pytest.mark.parametrize("missing", [False, True])
@pytest.mark.parametrize("T,w", SETTINGS)
@pytest.mark.parametrize("size", SIZES)
def test_cpu(size, T, w, missing):
    run("cpu", size, T, w, missing)


def slices(z, ids, values, targets, vocab, T, w, cuts, scale):
    """Loss and gradient by way of the statistics of column slices, as a mesh row computes them."""
    parts = [z[:, a:b].contiguous() for a, b in zip(cuts, cuts[1:])]
    st = [F.distill_partial(p, ids, values, a, vocab, T, targets) for p, a in zip(parts, cuts)]
    gmax = torch.stack([s[:, 0] for s in st]).amax(0)
    total = sum(distill_rescale(s, gmax, T) for s in st)
    total[:, 0] = gmax
    got = [F.distill_grad(p, ids, values, a, vocab, scale, total, T, targets, w) for p, a in zip(parts, cuts)]
    for other in got[1:]:
        assert torch.equal(other[0], got[0][0])
    return got[0][0], torch.cat([g for _, g in got], 1)


@pytest.mark.parametrize("T,w", SETTINGS)
def test_cpu_slices(T, w):
    z, ids, values, targets = data(11, 203, 256, 9, True)
    got = slices(z, ids, values, targets, 203, T, w, [0, 64, 128, 208, 256], 0.5)
    check(got, definition(z, ids, values, targets, 203, T, w), 0.5)


def test_gradient_against_differences():
    """Central differences of the definition's loss in 64 bits against the formulation's gradient (fp32 logits: no rounding to bf16)."""
    z, ids, values, targets = data(2, 20, 24, 5)
    z = z.float()
    for T, w in SETTINGS:
        _, grad = F.distill_loss_grad(z, ids, values, 20, 1.0, temperature=T, targets=targets, hard_weight=w)
        for c in range(20):
            d = torch.zeros_like(z, dtype=torch.float64)
            d[:, c] = 1e-4
            up, down = (definition(z.double() + s * d, ids, values, targets, 20, T, w)[0] for s in (1, -1))
            assert ((up - down) / 2e-4 - grad[:, c].double()).abs().max() < 1e-5


def test_duplicates_and_ignored_rows():
    """An id that occurs twice takes both probabilities; a row without entries and label is zero whatever its logits are."""
    z, ids, values, targets = data(3, 50, 56, 6)
    ids[:, 3] = ids[:, 0]
    want = definition(z, ids, values, targets, 50, 2.0, 0.5)
    check(F.distill_loss_grad(z, ids, values, 50, 1.0, 2.0, targets, 0.5), want, 1.0)
    z[1] = float("nan")
    ids[1], targets[1] = -1, -1
    loss, grad = F.distill_loss_grad(z, ids, values, 50, 1.0, 2.0, targets, 0.5)
    assert loss[1] == 0 and grad[1].count_nonzero() == 0 and torch.isfinite(grad).all()


def refusals(dev):
    z, ids, values, targets = (t.to(dev) for t in data(4, 50, 56, 6))
    ok = dict(vocab=50, scale=1.0)
    for args, kw in (((z, ids.int(), values), {}), ((z, ids[:2], values), {}), ((z, ids, values.double()), {}), ((z, ids, values[:, :3]), {}),
                     ((z, ids, values), dict(hard_weight=0.5)), ((z, ids, values), dict(hard_weight=1.5, targets=targets)),
                     ((z, ids, values), dict(temperature=0.0)), ((z, ids, values), dict(temperature=float("inf"))),
                     ((z, ids, values), dict(vocab=57)), ((z, ids, values), dict(vocab=0)), ((z, ids, values), dict(targets=targets.int())),
                     ((z, ids, values), dict(targets=targets[:2])), ((z[0], ids, values), {}), ((z, ids, values), dict(out=z.float()))):
        with pytest.raises(ValueError):
            F.distill_loss_grad(*args, **{**ok, **kw})
    with pytest.raises(ValueError):
        F.distill_grad(z, ids, values, 0, 50, 1.0, torch.zeros(4, 3, device=dev))
    with pytest.raises(ValueError):
        F.distill_partial(z, ids, values, -8, 50)


def test_refusals():
    refusals("cpu")


# ---------------------------------------------------------------------------------------------- on a GPU
@pytest.mark.gpu
@pytest.mark.parametrize("missing", [False, True])
@pytest.mark.parametrize("T,w", SETTINGS)
@pytest.mark.parametrize("size", SIZES + [(7, 5003, 5008, 128), (3, 30011, 30016, 64)])
def test_kernel(size, T, w, missing):
    run("cuda", size, T, w, missing)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(in_place=True), dict(values_dtype=torch.bfloat16), dict(use_targets=False)])
def test_kernel_forms(kw):
    for size in ((9, 1003, 1008, 20), (2, 110001, 110008, 5)):
        for T, w in ((1.0, 0.0), (2.0, 0.0)) if "use_targets" in kw else ((1.0, 0.5), (3.0, 0.5)):
            run("cuda", size, T, w, True, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("T,w", SETTINGS)
def test_kernel_slices(T, w):
    z, ids, values, targets = (t.cuda() for t in data(11, 2003, 2048, 37, True))
    want = definition(*(t.cpu() for t in (z, ids, values, targets)), 2003, T, w)
    check(slices(z, ids, values, targets, 2003, T, w, [0, 512, 1024, 2008, 2048], 0.5), want, 0.5)
    check(slices(z, ids, values, targets, 2003, T, w, [0, 2048], 0.5), want, 0.5)


@pytest.mark.gpu
def test_kernel_many_entries_and_duplicates():
    z, ids, values, targets = data(3, 3000, 3000, 1024)
    ids[:, 900:] = ids[:, 100:224]
    want = definition(z, ids, values, targets, 3000, 1.5, 0.2)
    a = [t.cuda() for t in (z, ids, values, targets)]
    got = F.distill_loss_grad(a[0], a[1], a[2], 3000, 1.0, 1.5, a[3], 0.2)
    check(got, want, 1.0)
    again = F.distill_loss_grad(a[0], a[1], a[2], 3000, 1.0, 1.5, a[3], 0.2)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.gpu
def test_kernel_ignored_rows_infinities_and_nan():
    """Rows that nothing is learnt from are zero; -inf logits have probability 0; a NaN shows in its own row alone."""
    for vocab in (1000, 104000):
        z, ids, values, targets = (t.cuda() for t in data(6, vocab, vocab, 6))
        z[0] = float("nan")
        ids[0], targets[0] = -1, -1
        z[1, 100:] = -math.inf
        ids[1], targets[1] = torch.arange(6, device="cuda"), 7
        z[2, 5] = float("nan")
        values[3, 2] = float("nan")
        want = definition(*(t[[1, 4, 5]].cpu() for t in (z, ids, values, targets)), vocab, 2.0, 0.5)
        loss, grad = F.distill_loss_grad(z, ids, values, vocab, 1.0, 2.0, targets, 0.5)
        assert loss[0] == 0 and grad[0].count_nonzero() == 0
        check((loss[[1, 4, 5]], grad[[1, 4, 5]]), want, 1.0)
        assert grad[1, 100:].count_nonzero() == 0
        assert loss[2].isnan() and loss[3].isnan() and grad[2].isnan().any() and grad[3].isnan().any()


@pytest.mark.gpu
def test_kernel_strides_and_alignment():
    z, ids, values, targets = (t.cuda() for t in data(7, 203, 208, 9, True))
    a = (203, 0.5, 2.0, targets, 0.5)
    want = F.distill_loss_grad(z, ids, values, *a)
    wide = torch.zeros(7, 240, dtype=torch.bfloat16, device="cuda")
    for at in (0, 8, 3):
        cut = wide[:, at:at + 208].copy_(z)
        got = F.distill_loss_grad(cut, ids.T.contiguous().T, values.T.contiguous().T, *a)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for to in (0, 16, 1):
            out = torch.zeros(7, 250, dtype=torch.bfloat16, device="cuda")
            got = F.distill_loss_grad(cut, ids, values, *a, out=out[:, to:to + 208])
            assert torch.equal(got[1], want[1]) and torch.equal(out[:, to:to + 208], want[1])
            assert out[:, :to].count_nonzero() == 0 and out[:, to + 208:].count_nonzero() == 0
        got = F.distill_loss_grad(cut, ids, values, *a, out=cut)
        assert torch.equal(cut, want[1])
    block = torch.zeros(8, 208, dtype=torch.bfloat16, device="cuda")
    block[:7].copy_(z)
    assert torch.equal(F.distill_loss_grad(block[:7], ids, values, *a, out=block[1:])[1], want[1])
    empty = F.distill_loss_grad(z[:0], ids[:0], values[:0], 203, 0.5, 2.0, targets[:0], 0.5)
    assert empty[0].shape == (0,) and empty[1].shape == (0, 208)


@pytest.mark.gpu
def test_kernel_refusals():
    refusals("cuda")
    z, ids, values, _ = (t.cuda() for t in data(4, 50, 56, 6))
    with pytest.raises(ValueError):
        F.distill_loss_grad(z.float(), ids, values, 50, 1.0)
    with pytest.raises(ValueError):
        F.distill_loss_grad(z[:, :51], ids, values, 50, 1.0)
    with pytest.raises(ValueError):
        F.distill_loss_grad(z, ids.cpu(), values, 50, 1.0)
    with pytest.raises(ValueError):
        F.distill_loss_grad(z, ids.repeat(1, 200), values.repeat(1, 200), 50, 1.0)


LOWEST = torch.finfo(torch.bfloat16).min
FILLS = [LOWEST, -1e30, -1e10, -1e4]


def masked(dev, vocab, fill, T, w, how):
    """Logits that a mask has filled: a run of columns longer than what a thread sums at a time, a few, all of a row, all but one; and one
    that is as far above the others.  The teacher's entries and the label are beside the mask, in the third row inside it."""
    n, cols, top = 5, -(-vocab // 8) * 8, 6
    z, ids, values, targets = data(n, vocab, cols, top, seed=3)
    ids = vocab - 1 - torch.arange(top).repeat(n, 1) * max(1, vocab // 40)
    targets = ids[:, 2].clone()
    z[0, : vocab * 3 // 4] = fill
    z[1, 8:40] = fill
    z[2] = fill
    z[3] = fill
    z[3, vocab - 1] = 1.5
    ids[3], targets[3] = torch.tensor([vocab - 1] + [-1] * (top - 1)), vocab - 1
    z[4, 3] = -fill
    ids[4], targets[4] = torch.tensor([3] + [-1] * (top - 1)), 3
    want = definition(z, ids, values, targets, vocab, T, w)
    a = [t.to(dev) for t in (z, ids, values, targets)]
    got = how(a, vocab, T, w)
    assert got[0].isfinite().all() and got[1].isfinite().all()
    check(got, want, 0.5)
    # beyond 2^24 T not by the size of the logits, but by that of their differences (below, sums of p z are rounded to their own size)
    for r in (2, 3, 4) if abs(fill) >= 2.0 ** 24 * T else ():
        p = torch.softmax(values[r][(ids[r] >= 0)].double() / T, 0)
        rest = math.log(vocab) + 1 + (p * p.log()).sum().abs()
        assert abs(got[0][r].double().cpu() - want[0][r]) <= 2.0 ** -19 * ((1 - w) * T * T + w) * rest


WAYS = {"rows": lambda a, vocab, T, w: F.distill_loss_grad(a[0], a[1], a[2], vocab, 0.5, T, a[3], w),
        "slices": lambda a, vocab, T, w: slices(*a, vocab, T, w, [0, vocab // 32 * 8, vocab // 16 * 8, a[0].shape[1]], 0.5)}


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("T,w", SETTINGS)
@pytest.mark.parametrize("fill", FILLS)
def test_cpu_masked_logits(fill, T, w, way):
    masked("cpu", 203, fill, T, w, WAYS[way])


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,way", [(203, "rows"), (6000, "rows"), (30011, "rows"), (104000, "rows"), (6000, "slices")])
@pytest.mark.parametrize("T,w", SETTINGS + [(3.0, 0.5), (40.0, 0.5)])
@pytest.mark.parametrize("fill", FILLS)
def test_kernel_masked_logits(fill, T, w, vocab, way):
    masked("cuda", vocab, fill, T, w, WAYS[way])


def dense(z, ids, values, targets, vocab, T, w):
    """``definition`` for many rows at a time, on the tensors' device; every id occurs once."""
    x, n = z[:, :vocab].double(), z.shape[0]
    there = (ids >= 0) & (ids < vocab) & (values.float() != -math.inf)
    r, k = there.nonzero(as_tuple=True)
    t = torch.full_like(x, -math.inf)
    t[r, ids[r, k]] = values[r, k].double()
    p = torch.softmax(t / T, 1).nan_to_num_(0.0)                       # (rows without entries)
    some = there.any(1)
    plogp = (p * p.clamp_min(1e-300).log()).sum(1)
    logq, m, far = torch.log_softmax(x / T, 1), x.amax(1), (x - x.amax(1, keepdim=True)).abs()
    loss = torch.where(some, (1 - w) * T * T * (plogp - (p * logq).sum(1)), 0.0)
    parts_of_loss = T * T * (1 + plogp.abs() + torch.logsumexp(x / T, 1).abs() + m.abs()) + T * (p * far).sum(1)
    size = 1 + torch.where(some, parts_of_loss if w != 1.0 else 0.0, 0.0)
    q = logq.exp_() * some[:, None] * ((1 - w) * T)
    grad, parts = q - (1 - w) * T * p, q + (1 - w) * T * p
    label = ((targets >= 0) & (targets < vocab)).nonzero()[:, 0]
    y = targets[label]
    if w != 0.0:
        logq = torch.log_softmax(x, 1)
        loss[label] -= w * logq[label, y]
        size[label] += torch.logsumexp(x, 1)[label].abs() + far[label, y] + m[label].abs()
        hard = torch.zeros_like(x)
        hard[label] = w * logq[label].exp()
        grad += hard
        parts += hard
        grad[label, y] -= w
        parts[label, y] += w
    pad = lambda v: torch.nn.functional.pad(v, (0, z.shape[1] - vocab)).cpu()
    return loss.cpu(), pad(grad), size.cpu(), pad(parts)


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("T,w", [(1.0, 0.3), (0.7, 1.0), (2.0, 0.5), (4.0, 0.1), (3.0, 0.5)])
@pytest.mark.parametrize("rows,vocab,top", [(3200, 1003, 9), (1100, 8200, 200), (900, 12003, 20), (700, 45007, 33), (450, 60001, 64)])
def test_kernel_rows_of_a_cta_follow_one_another(rows, vocab, top, T, w, in_place):
    """Two to four rows for every CTA that is resident, of each width: entries, labels, neither and NaN by turns.  Every row is what it is
    among a few others, bit by bit, and what the definition says."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    cols = -(-vocab // 16) * 16
    z = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16).normal_(0, 2, generator=g)
    values, ids = torch.rand(rows, vocab, device="cuda", generator=g).topk(top, 1)
    values = (values - 0.9) * 40 + torch.empty_like(values).normal_(0, 3, generator=g)
    targets = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    targets[::2] = ids[::2, 0]
    of = torch.randint(0, 6, (rows,), device="cuda", generator=g)      # 0, 1: all; 2: no label; 3: no entry; 4: some entries; 5: neither
    targets[(of == 2) | (of == 5)] = -1
    ids[(of == 3) | (of == 5)] = -1
    ids[of == 4, top // 2:] = vocab
    nan = (of == 5) & (torch.arange(rows, device="cuda") % 2 == 0)
    z[nan] = float("nan")
    a = (ids, values, vocab, 0.25, T, targets, w)
    few = [F.distill_loss_grad(z[i:i + 90], ids[i:i + 90], values[i:i + 90], vocab, 0.25, T, targets[i:i + 90], w) for i in range(0, rows, 90)]
    x = z.clone() if in_place else z
    loss, grad = F.distill_loss_grad(x, *a, out=x if in_place else None)
    assert torch.equal(loss, torch.cat([l for l, _ in few])) and torch.equal(grad, torch.cat([g for _, g in few]))
    assert loss[of == 5].count_nonzero() == 0 and grad[of == 5].count_nonzero() == 0 and grad[:, vocab:].count_nonzero() == 0
    check((loss, grad), dense(z.masked_fill(nan[:, None], 0.0), ids, values, targets, vocab, T, w), 0.25)


@pytest.mark.gpu
def test_kernel_on_another_stream_and_in_a_graph():
    z, ids, values, targets = (t.cuda() for t in data(2500, 1003, 1008, 9, True))
    a = (1003, 0.5, 2.0, targets, 0.5)
    want = F.distill_loss_grad(z, ids, values, *a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = z.clone().mul_(1)
        got = F.distill_loss_grad(x, ids, values, *a, out=x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(x, want[1])
    x = torch.zeros_like(z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = F.distill_loss_grad(x, ids, values, *a)
        stats = F.distill_partial(x, ids, values, 0, 1003, 2.0, targets)
        by_slices = F.distill_grad(x, ids, values, 0, 1003, 0.5, stats, 2.0, targets, 0.5)
    for _ in range(2):
        x.copy_(z)
        graph.replay()
        assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])
        assert torch.allclose(by_slices[0], loss, rtol=1e-4, atol=1e-4) and torch.allclose(by_slices[1].float(), grad.float(), rtol=2 ** -6, atol=2.5e-5)
        x.zero_()


def shared_ids(dev):
    """Entries of one id against one entry of their joint probability: the same gradient, and a loss that differs by what they are
    uncertain among themselves, whatever the logits are."""
    z, ids, values, targets = data(6, 203, 208, 4, seed=9)
    for T, w in ((1.0, 0.0), (2.0, 0.5), (3.0, 0.3)):
        twice = torch.cat([ids, ids[:, :1], ids[:, :2]], 1)
        more = torch.cat([values, values[:, :1] + 0.5, values[:, :2] - 1.0], 1)
        p = torch.softmax(more.double() / T, 1)
        joint = p[:, :4].clone()
        joint[:, 0] += p[:, 4] + p[:, 5]
        joint[:, 1] += p[:, 6]
        among = (joint * joint.log()).sum(1) - (p * p.log()).sum(1)
        assert (among > 0).all() and among.max() > 0.1
        for x in (z, (z.float() * 0.3 + 1.0).bfloat16()):
            a = [t.to(dev) for t in (x, twice, more, targets, ids, (T * joint.log()).float())]
            loss, grad = F.distill_loss_grad(a[0], a[1], a[2], 203, 1.0, T, a[3], w)
            one, same = F.distill_loss_grad(a[0], a[4], a[5], 203, 1.0, T, a[3], w)
            assert ((one - loss).double().cpu() - (1 - w) * T * T * among).abs().max() < 1e-4
            # (p of either is rounded to 24 bits, the gradient to bf16)
            assert ((grad - same).float().abs() <= 2.0 ** -7 * same.float().abs() + 1e-5).all()


def test_cpu_entries_that_share_an_id():
    shared_ids("cpu")


@pytest.mark.gpu
def test_kernel_entries_that_share_an_id():
    shared_ids("cuda")
