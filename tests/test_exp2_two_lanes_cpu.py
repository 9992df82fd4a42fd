"""The two-lane exponential of the window attention's backward kernel, restated in fp32 from the constants in its source."""
import re
from pathlib import Path

import numpy as np

SOURCE = Path(__file__).resolve().parent.parent / "meshslice_b200" / "csrc" / "ops" / "window_attention.cu"


def _exp2_poly(x):
    body = re.search(r"void exp2_poly\(uint64_t x, float& a, float& b\) \{(.*?)\n\}", SOURCE.read_text(), re.S).group(1)
    first = np.float32(re.search(r"uint64_t p = f32x2\(([0-9.e+-]+)f,", body).group(1))
    coefs = [np.float32(c) for c in re.findall(r"p = fma2\(p, f, f32x2\(([0-9.e+-]+)f,", body)]
    assert len(coefs) == 5
    # the last step: times the power of two that the low bits of r stand for
    assert "mul2(p, f32x2(__int_as_float((__float_as_int(a) << 23) + 0x3f800000)" in body
    x = np.asarray(x, np.float32)
    t = np.where(np.isnan(x), x, np.maximum(x, np.float32(-125)))
    r = t + np.float32(12582912)
    f = t - (r - np.float32(12582912))
    p = np.full_like(f, first)
    for c in coefs:                        # one rounding per step: the product of two fp32 is exact in fp64
        p = (p.astype(np.float64) * f + np.float64(c)).astype(np.float32)
    scale = ((r.view(np.int32) << 23) + 0x3F800000).astype(np.int32).view(np.float32)
    return p * scale


def test_two_lane_polynomial_is_as_accurate_as_the_instruction_beside_it():
    """As for the one-lane form: relative error against 64 bits at most 2^-22 up to 126, 2^-125 below -125, NaN stays NaN (with every
    payload and sign)."""
    g = np.random.default_rng(1)
    x = np.concatenate([g.uniform(-125, 0, 1 << 20), g.uniform(-2, 2, 1 << 20), g.uniform(0, 126, 1 << 18),
                        np.arange(-125, 127), np.arange(-124.5, 126)]).astype(np.float32)
    assert np.max(np.abs(_exp2_poly(x) / np.exp2(x.astype(np.float64)) - 1)) <= 2.0 ** -22
    low = _exp2_poly(np.array([-125.0, -125.5, -126, -1000, -1e30, -np.inf], np.float32))
    assert np.all(np.abs(low / 2.0 ** -125 - 1) <= 2.0 ** -22)
    assert np.all(np.isnan(_exp2_poly(np.array([0x7fffffff, 0x7fc00000, 0xffc00000, 0xffffffff], np.uint32).view(np.float32))))
