"""Single tokens over the ring cache: CPU formulation and kernel against dense attention over the whole history in 64 bits."""
import math

import pytest
import torch

from meshslice_b200.ops import functional as F
from meshslice_b200.ops.window import WindowCache


def history(batch, length, kv, group, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(batch, length, kv, group + 2, D, generator=g).bfloat16()


def definition(x, p, window, sinks):
    """Output of position p of one sequence [length, kv, group + 2, D] in 64 bits, from all positions up to p."""
    g = x.shape[2] - 2
    j = torch.arange(p + 1)
    seen = j[(p - j < window) | (j < sinks)]
    q, k, v = x[p, :, :g].double(), x[seen, :, g].double(), x[seen, :, g + 1].double()
    w = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(x.shape[3]), -1)
    return torch.einsum("hgn,nhd->hgd", w, v).reshape(-1), v.abs().max()


def check(got, want, vmax):
    """P is rounded to bf16 (2^-8 of each probability, whose sum is 1) and so is the result: 2^-7 of the largest value at most; the
    scores' fp32 rounding and the exponentials are below 2^-12 of it."""
    assert ((got.double().cpu() - want).abs() <= (2.0 ** -7 + 2.0 ** -12) * vmax).all()


SIZES = [(3, 2, 1, 5, 0), (2, 1, 3, 1, 0), (2, 2, 8, 16, 4), (3, 1, 16, 37, 1), (1, 3, 2, 64, 20), (2, 1, 17, 9, 2), (2, 1, 40, 30, 3)]


@pytest.mark.parametrize("size", SIZES)
def test_cpu_token_by_token(size):
    batch, kv, group, window, sinks = size
    n, D = 2 * window + sinks + 7, 32
    x = history(batch, n, kv, group, D)
    cache = WindowCache.new(batch, kv, window, sinks, head_dim=D)
    for p in range(n):
        got = F.window_attention_decode(x[:, p].reshape(batch, -1), cache, torch.full((batch,), p), group)
        for b in range(batch):
            check(got[b], *definition(x[b], p, window, sinks))


@pytest.mark.parametrize("seq", [1, 3, 4, 5, 20, 21, 60])
def test_fill_is_token_by_token(seq):
    x = history(2, seq, 2, 3, 32)
    a, b = (WindowCache.new(2, 2, 17, 4, head_dim=32) for _ in range(2))
    a.fill(x.reshape(2 * seq, -1), seq, 3)
    for p in range(seq):
        F.window_attention_decode(x[:, p].reshape(2, -1), b, torch.full((2,), p), 3)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def refusals(dev):
    k = torch.zeros(2, 1, 6, 128, dtype=torch.bfloat16, device=dev)
    for args in ((k, k, 6, 1), (k, k[:1], 5, 1), (k, k.float(), 5, 1), (k, k, 0, 6), (k, k, 7, -1), (k[0], k[0], 5, 1)):
        with pytest.raises(ValueError):
            WindowCache(*args)
    cache, x, pos = WindowCache(k, k.clone(), 5, 1), torch.zeros(2, 3 * 128, dtype=torch.bfloat16, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    for args in ((x, cache, pos.int()), (x, cache, pos[:1]), (x[:1], cache, pos), (x, cache, pos, 2), (x, cache, pos, 0), (x.float(), cache, pos),
                 (x[:, :192], cache, pos)):
        with pytest.raises(ValueError):
            F.window_attention_decode(*args)
    with pytest.raises(ValueError):
        cache.fill(x, 2)
    with pytest.raises(AttributeError):
        cache.k = k


def test_refusals():
    refusals("cpu")


# ---------------------------------------------------------------------------------------------- on a GPU
@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES + [(2, 2, 4, 300, 4), (1, 1, 1, 2000, 0), (1, 1, 3, 6000, 5)])
def test_kernel(size):
    """Positions from the first to far beyond the window; every slot that holds nothing yet is NaN."""
    batch, kv, group, window, sinks = size
    n = 2 * window + sinks + 7
    x = history(batch, n, kv, group, 128)
    rows = x.view(batch, n, -1).cuda()
    nan = torch.full((batch, kv, window + sinks, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    cache = WindowCache(nan, nan.clone(), window, sinks)
    stops = sorted({0, 1, sinks, window - 1, window, window + sinks - 1, window + sinks, window + sinks + 1, n - 2, n - 1} & set(range(n)))
    for p in stops:
        if p:
            cache.fill(rows[:, :p].reshape(batch * p, -1), p, group)
        before = cache.k.clone(), cache.v.clone()
        got = F.window_attention_decode(rows[:, p].contiguous(), cache, torch.full((batch,), p, device="cuda"), group)
        for b in range(batch):
            check(got[b], *definition(x[b], p, window, sinks))
        slot = int(cache.slots(torch.tensor(p)))
        for t, old, i in ((cache.k, before[0], group), (cache.v, before[1], group + 1)):
            old[:, :, slot] = x[:, p, :, i].cuda()
            assert torch.equal(t.nan_to_num(9.0), old.nan_to_num(9.0))


@pytest.mark.gpu
def test_kernel_mixed_positions_idle_sequences_strides_and_repeats():
    batch, kv, group, window, sinks = 9, 2, 4, 200, 4
    stops = [0, 5, -1, 203, 204, 399, -7, 1, 60]
    x = history(batch, 400, kv, group, 128)
    cache = WindowCache.new(batch, kv, window, sinks, device="cuda")
    for b, p in enumerate(stops):
        if p > 0:
            one = WindowCache.new(1, kv, window, sinks, device="cuda")
            one.fill(x[b, :p].reshape(p, -1).cuda(), p, group)
            cache.k[b], cache.v[b] = one.k[0], one.v[0]
    rows = torch.stack([x[b, max(p, 0)].reshape(-1) for b, p in enumerate(stops)]).cuda()
    pos = torch.tensor(stops, device="cuda")
    idle = [b for b, p in enumerate(stops) if p < 0]
    old = cache.k[idle].clone()
    got = F.window_attention_decode(rows, cache, pos, group)
    for b, p in enumerate(stops):
        if p < 0:
            assert got[b].count_nonzero() == 0
        else:
            check(got[b], *definition(x[b], p, window, sinks))
    assert torch.equal(cache.k[idle], old)
    wide = torch.zeros(batch, rows.shape[1] + 24, dtype=torch.bfloat16, device="cuda")
    for at in (0, 8, 3):
        cut = wide[:, at:at + rows.shape[1]].copy_(rows)
        assert torch.equal(F.window_attention_decode(cut, cache, torch.stack([pos, pos], 1)[:, 0], group), got)


@pytest.mark.gpu
def test_kernel_large_cache_beyond_32_bits():
    """More than 2^32 elements: offsets of the last sequences need 64 bits."""
    batch, kv, window = 9, 4, 1 << 20
    cache = WindowCache(*(torch.empty(batch, kv, window, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)), window, 0)
    assert cache.k.numel() > 2 ** 32
    x = history(batch, 3, kv, 2, 128)
    for p in range(3):
        got = F.window_attention_decode(x[:, p].reshape(batch, -1).cuda(), cache, torch.full((batch,), p, device="cuda"), 2)
    for b in (0, batch - 1):
        check(got[b], *definition(x[b], 2, window, 0))
    assert torch.equal(cache.k[-1, -1, 2].cpu(), x[-1, 2, -1, 2])


@pytest.mark.gpu
def test_kernel_in_a_graph_and_refusals():
    refusals("cuda")
    x = history(4, 50, 2, 2, 128)
    cache = WindowCache.new(4, 2, 30, 2, device="cuda")
    rows, pos = torch.zeros(4, 2 * 4 * 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.window_attention_decode(rows, cache, pos - 1, 2)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.window_attention_decode(rows, cache, pos, 2)
    for p in range(50):
        rows.copy_(x[:, p].reshape(4, -1))
        pos.fill_(p)
        graph.replay()
        for b in range(4):
            check(out[b], *definition(x[b], p, 30, 2))
    with pytest.raises(ValueError):
        WindowCache(cache.k.transpose(0, 1), cache.v.transpose(0, 1), 30, 2)
    with pytest.raises(ValueError):
        WindowCache.new(1, 1, 4, head_dim=64, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("group", [3, 12])
@pytest.mark.parametrize("batch,window", [(1, 700), (40, 700), (1, 20000)])
def test_kernel_keys_of_minus_infinity(batch, window, group):
    """Keys whose score is -inf have probability 0, also where a warp's first tiles, or all of a split, have no other."""
    n = window + 1
    x = history(1, n, 1, group, 128)
    x[..., :group, 0] = 1.0
    x[:, 1:window // 2, :, group, 0] = -math.inf
    cache = WindowCache.new(batch, 1, window, 0, device="cuda")
    cache.fill(x[0, : n - 1].reshape(n - 1, -1).repeat(batch, 1).cuda(), n - 1, group)
    got = F.window_attention_decode(x[:, n - 1].reshape(1, -1).repeat(batch, 1).cuda(), cache, torch.full((batch,), n - 1, device="cuda"), group)
    assert torch.equal(got, got[:1].expand_as(got))
    check(got[0], *definition(x[0], n - 1, window, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2900, 7000])
def test_kernel_whose_first_call_is_captured(window):
    """The workspace that a graph lays out is the graph's own: calls outside of it, before its first run too, are right."""
    x = history(1, window + 100, 1, 2, 128)
    cache = WindowCache.new(1, 1, window, 2, device="cuda")
    cache.fill(x[0, :window + 99].reshape(window + 99, -1).cuda(), window + 99, 2)
    row, pos = x[:, window + 99].reshape(1, -1).cuda(), torch.full((1,), window + 99, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.window_attention_decode(row, cache, pos, 2)
    want = definition(x[0], window + 99, window, 2)
    check(F.window_attention_decode(row, cache, pos, 2)[0], *want)
    for _ in range(2):
        graph.replay()
        check(out[0], *want)
    del graph
    check(F.window_attention_decode(row, cache, pos, 2)[0], *want)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 4), (1, 8), (1, 11), (1, 33)])
@pytest.mark.parametrize("window", [190, 250, 400, 1000, 1400, 1600, 7000])
def test_kernel_splits_that_hold_nothing_yet(kv, group, window):
    """Sequences of every number of splits in use, up to all of them, beside one another."""
    stops = [0, -1, window - 1] + list(range(63, 2 * window, window // 7 + 1))
    x = history(1, 2 * window, kv, group, 128)
    rows = x[0, [max(p, 0) for p in stops]].reshape(len(stops), -1).cuda()
    cache = WindowCache.new(len(stops), kv, window, 3, device="cuda")
    whole = x[0].reshape(2 * window, -1).cuda()
    for b, p in enumerate(stops):
        if p > 0:
            one = WindowCache.new(1, kv, window, 3, device="cuda")
            one.fill(whole[:p], p, group)
            cache.k[b], cache.v[b] = one.k[0], one.v[0]
    got = F.window_attention_decode(rows, cache, torch.tensor(stops, device="cuda"), group)
    for b, p in enumerate(stops):
        if p < 0:
            assert got[b].count_nonzero() == 0
        else:
            check(got[b], *definition(x[0], p, window, 3))


def test_sizes_without_heads_sequences_or_slots():
    """The sizes that a launch lays out are worked out before anything checks its arguments: nothing to deal out is an answer, and no
    division by it; a cache without heads or features is refused."""
    from meshslice_b200 import _native
    C = _native.load()
    for args in ((1, 0, 1, 8, 148), (0, 4, 1, 8, 148), (1, 4, 0, 8, 148), (1, 4, 1, 0, 148), (1, -1, 1, 8, 148), (1, 4, 1, 8, 0)):
        assert C.window_decode_splits(*args) == 1
    assert C.window_decode_splits(1, 1, 1, 131072, 148) > 8
    for batch, kv in ((0, 1), (1, 0), (0, 0), (-1, 1)):
        assert C.window_attention_scratch(batch, 200, kv, 1, 64, 4) <= 0
    assert C.window_attention_scratch(1, 200, 1, 1, 64, 4) > 0
    for shape in ((2, 0, 6, 128), (2, 1, 6, 0)):
        k = torch.zeros(shape, dtype=torch.bfloat16)
        with pytest.raises(ValueError):
            WindowCache(k, k.clone(), 5, 1)
    with pytest.raises(ValueError):
        WindowCache.new(2, 0, 5, 1)
