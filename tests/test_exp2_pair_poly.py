"""The FMA-pipe exponential of the attention-weight kernels (fast_math.cuh, exp2_2_poly), on the CPU.

One pair of scores in eight goes through n = round(x), f = x - n and a degree-5 polynomial for
2^f, n added to the exponent field.  This restates those steps in numpy with the constants
read from the source, and checks the errors that the source states: those of the stored
coefficients in 64 bits, those of the float32 evaluation, and the values at the ends.
"""
import os
import re

import numpy as np

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "smol-genius_b200", "csrc",
                   "fast_math.cuh")
TEXT = open(SRC).read()


def _coefficients():
    body = TEXT.split("f32x2 exp2_2_poly(f32x2 x)", 1)[1].split("\n}\n", 1)[0]
    c = [float.fromhex(x) for x in re.findall(r"both\((0x1[0-9a-f.]*p[-+]\d+)f\)", body)]
    assert len(c) == 6, body
    assert all(float(np.float32(x)) == x for x in c)
    return c


def _clamp_ends():
    body = TEXT.split("float clamp_exp(float x)", 1)[1].split("\n}\n", 1)[0]
    return [np.array([int(x, 16)], np.uint32).view(np.float32)[0] for x in re.findall(r"0f([0-9A-F]{8})", body)]


def exp2_pair_poly(x):
    f32 = np.float32
    lo, hi = _clamp_ends()
    x = np.minimum(np.maximum(x.astype(f32), lo), hi)    # numpy keeps NaN here, as max.NaN / min.NaN do
    magic = f32(12582912.0)
    j = (x + magic).astype(f32)
    f = (x - (j - magic).astype(f32)).astype(f32).astype(np.float64)
    c = _coefficients()
    p = np.full_like(x, f32(c[0]))
    for a in c[1:]:   # fused multiply-adds: one rounding each
        p = (p.astype(np.float64) * f + a).astype(f32)
    # NaN as the GPU's arithmetic gives it: 0x7fffffff
    pb = np.where(np.isnan(p), np.uint32(0x7fffffff), p.view(np.uint32))
    jb = np.where(np.isnan(j), np.uint32(0x7fffffff), j.view(np.uint32))
    with np.errstate(over="ignore"):
        return (pb + (jb << np.uint32(23))).astype(np.uint32).view(f32)


def test_stored_coefficients_in_64_bits():
    f = np.linspace(-0.5, 0.5, 1_000_001)
    rel = np.abs(np.polyval(_coefficients(), f) / np.exp2(f) - 1)
    assert 1.50e-7 < rel.max() < 1.56e-7, rel.max()


def test_coefficients_are_the_minimax_fit():
    x = np.cos(np.pi * (np.arange(2000) + 0.5) / 2000) / 2
    a = np.vander(x, 6) / np.exp2(x)[:, None]
    w = np.ones_like(x)
    for _ in range(1000):     # Lawson: weights grow with the error they leave
        c = np.linalg.lstsq(a * np.sqrt(w)[:, None], np.sqrt(w), rcond=None)[0]
        e = np.abs(a @ c - 1)
        w = w * e / (w * e).sum()
    assert e.max() < 7.55e-8
    for got, want in zip(_coefficients(), c):
        assert abs(got - want) <= 4e-6 * abs(want) + 2.0 ** -24


def test_float32_evaluation():
    x = np.linspace(-125.9, 126.9, 2_000_001, dtype=np.float32)
    rel = np.abs(exp2_pair_poly(x).astype(np.float64) / np.exp2(x.astype(np.float64)) - 1)
    assert rel.max() < 2.2e-7, rel.max()


def test_ends_and_special_values():
    assert _clamp_ends() == [-126.0, 127.0]
    least = exp2_pair_poly(np.array([-126.0, -126.5, -1e30, -np.inf], np.float32))
    assert np.all(least == least[0]) and abs(float(least[0]) * 2.0 ** 126 - 1) < 2e-7
    most = exp2_pair_poly(np.array([127.0, 1e30, np.inf], np.float32))
    assert np.all(most == most[0]) and np.isfinite(most[0]) and most[0] > 2.0 ** 126
    nan = exp2_pair_poly(np.array([np.nan], np.float32))
    assert nan[0] == np.finfo(np.float32).max       # above every sum of probabilities: the caller looks again
