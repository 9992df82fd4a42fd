"""Rotary positions: the CPU formulation and the kernel against the definition in 64 bits."""
import cmath
import math

import pytest
import torch

from meshslice_b200.ops import functional as F
from meshslice_b200.ops.rotary import Rotary, RotaryConfig


def definition(x, freq, m, layout, rot, kv, group, positions, inverse):
    """Pair by pair, a complex product in 64 bits."""
    tokens, D = x.shape[0], x.shape[1] // (kv * (group + 2))
    y = x.double().view(tokens, kv, group + 2, D).clone()
    i = torch.arange(rot // 2)
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    angle = positions.double()[:, None] * torch.tensor(freq, dtype=torch.float64) * (-1 if inverse else 1)
    c, s = angle.cos()[:, None, None] * m, angle.sin()[:, None, None] * m
    qk = y[:, :, :-1]
    u, v = qk[..., a], qk[..., b]
    y[:, :, :-1, a] = u * c - v * s
    y[:, :, :-1, b] = v * c + u * s
    return y.view(tokens, -1)


def rows(tokens, kv, group, D, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(tokens, kv * (group + 2) * D, generator=g).to(dtype)


def off_by(got, want, m):
    """Largest error in units of what it may be: half a unit in the last of bf16's 8 bits, at most 2^-8 of the result, and 2^-20 of
    the largest one for fp32 products, their sum and the angle (2^-25 of a turn)."""
    length = want.abs().max().item()
    return ((got.double() - want).abs() / (2.0 ** -8 * want.abs() + 2.0 ** -20 * max(length, 1.0))).max().item()


SHAPES = [(1, 1, 1, 128, 128), (7, 2, 3, 128, 64), (33, 1, 8, 128, 96), (5, 3, 1, 64, 32), (300, 2, 4, 128, 128), (9, 1, 2, 256, 256),
          (4, 5, 2, 32, 16)]


def test_frequencies():
    """By their definitions: 'linear' divides all, 'base' keeps the first and divides the last, 'by_parts' keeps what turns fast and
    divides what turns less than once."""
    f = RotaryConfig(head_dim=128).frequencies()
    assert f[0] == 1.0 and abs(f[63] - 10000 ** (-126 / 128)) < 1e-15
    assert RotaryConfig(head_dim=128, scaling="linear", factor=4.0).frequencies() == [v / 4 for v in f]
    b = RotaryConfig(head_dim=128, scaling="base", factor=4.0).frequencies()
    assert b[0] == 1.0 and abs(b[63] / (f[63] / 4) - 1) < 1e-12
    c = RotaryConfig(head_dim=128, scaling="by_parts", factor=8.0, original_len=2048)
    p = c.frequencies()
    for v, w in zip(f, p):
        turns = 2048 * v / (2 * math.pi)
        if turns >= 32:
            assert w == v
        elif turns <= 1:
            assert abs(w * 8 / v - 1) < 1e-12
        else:
            assert v / 8 < w < v
    assert abs(c.cos_factor - (1 + 0.1 * math.log(8))) < 1e-15
    assert RotaryConfig(scaling="by_parts", factor=8.0, attention_factor=1.5).cos_factor == 1.5


def test_turns_wrap_at_any_position():
    """position * turns mod 2^64 is the angle's part of a turn, to 2^-40, at positions where fp32 radians are whole turns off."""
    r = Rotary(RotaryConfig(head_dim=64, theta=500000.0))
    for pos in (1, 2 ** 20 + 1, 2 ** 31 + 7):
        for t, f in zip(r.turns.tolist(), r.config.frequencies()):
            part = (pos * t) % (1 << 64) / 2.0 ** 64
            z = cmath.exp(1j * math.fmod(pos * f, 2 * math.pi))
            assert abs(cmath.exp(2j * math.pi * part) - z) < pos * 2.0 ** -52 + 1e-12


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES)
def test_cpu(shape, layout, inverse):
    tokens, kv, group, D, rot = shape
    c = RotaryConfig(head_dim=D, rot_dim=rot, layout=layout, scaling="by_parts", factor=4.0, original_len=64)
    x, pos = rows(tokens, kv, group, D), torch.arange(tokens) % 11
    got = F.rotary_qkv(x, Rotary(c), kv, group, seq=11, inverse=inverse)
    want = definition(x, c.frequencies(), c.cos_factor, layout, rot, kv, group, pos, inverse)
    assert off_by(got, want, c.cos_factor) <= 1.0
    v = x.view(tokens, kv, group + 2, D)
    assert torch.equal(got.view(tokens, kv, group + 2, D)[:, :, -1], v[:, :, -1])


def test_gradient_against_differences():
    """d/dx of sum(w * rotate(x)) is rotate back of w: central differences of the (linear) formulation in 64 bits."""
    c = RotaryConfig(head_dim=32, rot_dim=16, layout="interleaved", scaling="linear", factor=3.0)
    x, w = (rows(3, 1, 2, 32, s, torch.float32) for s in (1, 2))
    grad = F.rotary_qkv(w, Rotary(c), 1, 2, seq=3, inverse=True)
    f = lambda t: (definition(t, c.frequencies(), 1.0, c.layout, 16, 1, 2, torch.arange(3), False) * w.double()).sum()
    for i in range(0, x.numel(), 7):
        d = torch.zeros_like(x, dtype=torch.float64).view(-1)
        d[i] = 0.5
        d = d.view_as(x)
        assert abs((f(x.double() + d) - f(x.double() - d)).item() - grad.view(-1)[i].item()) < 1e-5


def test_refusals():
    for bad in (dict(head_dim=24), dict(rot_dim=8), dict(head_dim=64, rot_dim=80), dict(layout="pairs"), dict(scaling="twice"),
                dict(theta=0.0), dict(scaling="linear", factor=float("inf")), dict(scaling="by_parts", beta_fast=1.0), dict(head_dim=512)):
        with pytest.raises(ValueError):
            RotaryConfig(**bad)
    r, x = Rotary(RotaryConfig()), rows(4, 1, 1, 128)
    for args, kw in (((x, r, 2), dict(seq=4)), ((x, r, 0), dict(seq=4)), ((x, r, 1, 2), dict(seq=4)), ((x, r, 1), {}), ((x, r, 1), dict(seq=0)),
                     ((x, r, 1), dict(positions=torch.arange(3))), ((x, r, 1), dict(positions=torch.arange(4).int())),
                     ((x, r, 1), dict(seq=4, out=x.float())), ((x, r, 1), dict(seq=4, out=x[:2]))):
        with pytest.raises(ValueError):
            F.rotary_qkv(*args, **kw)


# ---------------------------------------------------------------------------------------------- on a GPU
@pytest.mark.gpu
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES + [(2100, 3, 1, 128, 128), (5000, 1, 1, 32, 16)])
def test_kernel(shape, layout, inverse):
    tokens, kv, group, D, rot = shape
    c = RotaryConfig(head_dim=D, rot_dim=rot, layout=layout, scaling="by_parts", factor=4.0, original_len=64)
    x = rows(tokens, kv, group, D)
    g = torch.Generator().manual_seed(1)
    r = Rotary(c, device="cuda")
    for pos, kw in ((torch.arange(tokens) % 13, dict(seq=13)), (torch.randint(-5, 1 << 20, (tokens,), generator=g), None)):
        xc = x.cuda()
        kw = dict(positions=pos.cuda()) if kw is None else kw
        want = definition(x, c.frequencies(), c.cos_factor, layout, rot, kv, group, pos, inverse)
        got = F.rotary_qkv(xc, r, kv, group, inverse=inverse, **kw)
        assert off_by(got.cpu(), want, c.cos_factor) <= 1.0
        assert torch.equal(xc.cpu(), x)
        there = F.rotary_qkv(xc, r, kv, group, inverse=inverse, out=xc, **kw)
        assert there is xc and torch.equal(xc, got)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_kernel_strides_and_alignment(layout):
    """Column slices, rows that no 16-byte load can take, outputs of every such kind, and outputs that overlap their input."""
    r = Rotary(RotaryConfig(head_dim=64, layout=layout), device="cuda")
    n, w = 37, 2 * 4 * 64
    x = rows(n, 2, 2, 64).cuda()
    want = F.rotary_qkv(x, r, 2, 2, seq=n)
    wide = torch.zeros(n, w + 24, dtype=torch.bfloat16, device="cuda")
    for first in (0, 8, 3):
        cut = wide[:, first:first + w].copy_(x)
        assert torch.equal(F.rotary_qkv(cut, r, 2, 2, seq=n), want)
        for at in (0, 16, 5):
            out = torch.zeros(n, w + 40, dtype=torch.bfloat16, device="cuda")
            got = F.rotary_qkv(cut, r, 2, 2, seq=n, out=out[:, at:at + w])
            assert torch.equal(got, want) and out[:, :at].count_nonzero() == 0 and out[:, at + w:].count_nonzero() == 0
        assert torch.equal(F.rotary_qkv(cut, r, 2, 2, seq=n, out=cut), want)
    block = torch.zeros(n + 1, w, dtype=torch.bfloat16, device="cuda")
    block[:n].copy_(x)
    assert torch.equal(F.rotary_qkv(block[:n], r, 2, 2, seq=n, out=block[1:]), want)
    odd = torch.zeros(n * w + 1, dtype=torch.bfloat16, device="cuda")[1:].view(n, w).copy_(x)
    assert torch.equal(F.rotary_qkv(odd, r, 2, 2, seq=n, out=odd), want) and torch.equal(odd, want)
    pos = torch.arange(2 * n, device="cuda")[::2]
    assert torch.equal(F.rotary_qkv(x, r, 2, 2, positions=pos), F.rotary_qkv(x, r, 2, 2, positions=pos.clone()))
    assert F.rotary_qkv(x[:0], r, 2, 2, seq=n).shape == (0, w)


@pytest.mark.gpu
def test_kernel_on_another_stream_and_refusals():
    r = Rotary(RotaryConfig(), device="cuda")
    x = rows(50, 2, 1, 128).cuda()
    want = F.rotary_qkv(x, r, 2, seq=50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x.clone().mul_(1)
        got = F.rotary_qkv(y, r, 2, seq=50)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    with pytest.raises(ValueError):
        F.rotary_qkv(x.float(), r, 2, seq=50)
    with pytest.raises(ValueError):
        F.rotary_qkv(x, Rotary(RotaryConfig()), 2, seq=50)
    with pytest.raises(ValueError):
        F.rotary_qkv(x, r, 2, positions=torch.arange(50))


def length_beside_positions(dev):
    """With positions given the length of a sequence is not looked at, whatever it is and wherever the result goes."""
    x, pos = rows(5, 1, 2, 128).to(dev), torch.tensor([3, 0, 9, 70000, 2], device=dev)
    rot = Rotary(RotaryConfig(head_dim=128), device=dev)
    want = F.rotary_qkv(x, rot, 1, 2, positions=pos)
    for seq in (None, 0, -3, 7, 1 << 40):
        assert torch.equal(F.rotary_qkv(x, rot, 1, 2, seq=seq, positions=pos), want)
        y = x.clone()
        assert torch.equal(F.rotary_qkv(y, rot, 1, 2, seq=seq, positions=pos, out=y), want)


def test_length_beside_positions():
    length_beside_positions("cpu")


@pytest.mark.gpu
def test_kernel_length_beside_positions():
    length_beside_positions("cuda")
