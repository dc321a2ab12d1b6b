"""The tcgen05 attention's exponential on the FMA pipes, its steps taken one by one in FP32 on the host."""

import os
import re

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F = np.float32


def coefficients():
    """The polynomial's, highest first, and the lowest x, as the kernel's source has them."""
    with open(os.path.join(ROOT, "ppocr-rs_b200", "csrc", "kernels", "attention_tc.cu")) as f:
        body = re.search(r"float2 exp2_fma\(float2 x\) \{(.*?)\n\}", f.read(), re.S).group(1)
    low = np.array([int(re.search(r"max\.NaN\.f32 %0, %0, 0f([0-9A-F]{8})", body).group(1), 16)], np.uint32).view(F)[0]
    pairs = re.findall(r"make_float2\(([0-9.]+)f, ([0-9.]+)f\)", body)
    assert all(a == b for a, b in pairs) and float(pairs[0][0]) == 1.5 * 2 ** 23
    return [F(a) for a, _ in pairs[1:]], low


def fma(a, b, c):
    """a b + c in FP32: the product is exact in FP64, whose sum is rounded once more."""
    return (a.astype(np.float64) * np.asarray(b, np.float64) + np.asarray(c, np.float64)).astype(F)


def exp2_fma(x):
    c, low = coefficients()
    with np.errstate(all="ignore"):
        x = np.where(np.isnan(x), x, np.maximum(x, low)).astype(F)
        t = (x + F(12582912)).astype(F)
        f = (x - (t - F(12582912)).astype(F)).astype(F)
        y = fma(f, c[0], c[1])
        for next_one in c[2:]:
            y = fma(y, f, next_one)
    return (y.view(np.uint32) + (t.view(np.uint32) << np.uint32(23))).view(F)


def test_ordinary_exponents():
    x = np.concatenate([np.linspace(-126, 9, 500001), np.arange(-126, 10), np.arange(-126, 9) + 0.5]).astype(F)
    y = exp2_fma(x).astype(np.float64)
    assert np.abs(y / np.exp2(x.astype(np.float64)) - 1).max() < 3e-6


def test_nothing_below_the_least_exponent():
    x = np.array([-127, -127.25, -128, -150, -1e4, -2.0 ** 40, -3e38, -np.inf], F)
    assert (exp2_fma(x) == 0).all()
    x = np.linspace(-127, -126, 1001).astype(F)   # subnormal ones: between 0 and the least normal number
    y = exp2_fma(x)
    assert (y >= 0).all() and (y <= F(2.0 ** -126) * F(1.00001)).all()


def test_no_number_stays_none():
    assert np.isnan(exp2_fma(np.array([np.nan], F))).all()
