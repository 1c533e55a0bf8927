"""CPU tier: the codes and ranges of csrc/row_codes.hpp (compiled with g++), by
which the sampler's second launch selects: a token outside the range that it asked
for would be counted outside its tables; and the logarithm of min-p's border."""
import ctypes
import decimal
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "native", "row_codes_host.cpp")
LIB = os.path.join(HERE, "native", "librow_codes_host.so")
HDRS = [os.path.join(os.path.dirname(HERE), "cudaforge_amd", "csrc", f)
        for f in ("row_codes.hpp", "common.hpp")]

F32, BF16, FP16 = 0, 1, 2


@pytest.fixture(scope="module")
def codes():
    if not os.path.exists(LIB) or os.path.getmtime(LIB) < max(map(os.path.getmtime, [SRC] + HDRS)):
        subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", SRC, "-o", LIB], check=True)
    lib = ctypes.CDLL(LIB)
    lib.codes_of.restype = ctypes.c_uint32
    lib.codes_of.argtypes = [ctypes.c_int, ctypes.c_float]
    lib.codes_value.restype = ctypes.c_float
    lib.codes_value.argtypes = [ctypes.c_int, ctypes.c_uint32]
    lib.codes_log2.restype = ctypes.c_double
    lib.codes_log2.argtypes = [ctypes.c_double, ctypes.c_float]
    lib.codes_wrong.argtypes = [ctypes.c_int, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_void_p,
                                ctypes.c_int]
    return lib


def _values(kind):
    """Every value of a 16-bit type; of fp32 the ends of each exponent's range and
    what lies around 0, with either sign, and NaN and infinities."""
    half = np.arange(1 << 16, dtype=np.uint32)
    if kind == BF16:
        bits = half << 16
    elif kind == FP16:
        return half.astype(np.uint16).view(np.float16).astype(np.float32)
    else:
        mag = np.concatenate([(np.arange(256)[:, None] << 23) + d for d in (-2, -1, 0, 1, 2)]
                             + [np.arange(600)[:, None]]).ravel()
        mag = np.unique(np.clip(mag, 0, 0x7fffffff)).astype(np.uint32)
        bits = np.concatenate([mag, mag | np.uint32(1 << 31)])
    return np.ascontiguousarray(bits).view(np.float32)


def _borders(codes, kind):
    x = _values(kind)
    x = x[np.isfinite(x)]
    near = np.sort(np.unique(np.abs(x)))[:6]
    some = np.concatenate([near, -near, np.random.default_rng(kind).choice(x, 40),
                           [x.max(), x.min(), 1.0, -1.0]]).astype(np.float32)
    return sorted({codes.codes_of(kind, float(v)) for v in some})


@pytest.mark.parametrize("kind", [F32, BF16, FP16])
def test_codes_are_in_the_order_of_the_values(codes, kind):
    x = _values(kind)
    x = np.sort(x[np.isfinite(x)])
    got = np.array([codes.codes_of(kind, float(v)) for v in x[::7]], dtype=np.int64)
    assert (np.diff(got)[np.diff(x[::7]) > 0] > 0).all()
    for v in x[::7]:
        back = codes.codes_value(kind, codes.codes_of(kind, float(v)))
        assert back == v and np.signbit(back) == np.signbit(v)
    # both zeros have one: -0's is the one in front of 0's
    assert codes.codes_of(kind, -0.0) + 1 == codes.codes_of(kind, 0.0)


@pytest.mark.parametrize("kind", [F32, BF16, FP16])
def test_a_range_holds_its_codes_alone(codes, kind):
    """Every pair of borders, the two zeros' and the least values' around them
    among them: -0 as an upper border let +0 in, whose code is one more."""
    x = np.ascontiguousarray(_values(kind))
    at = _borders(codes, kind)
    assert codes.codes_of(kind, -0.0) in at
    for i, lo in enumerate(at):
        for hi in at[i:]:
            assert codes.codes_wrong(kind, lo, hi, x.ctypes.data, len(x)) == 0, (hex(lo), hex(hi))


@pytest.mark.parametrize("kind", [F32, BF16, FP16])
def test_the_range_of_minus_zero_alone_is_empty(codes, kind):
    zero = np.array([0.0, -0.0], dtype=np.float32)
    c = codes.codes_of(kind, -0.0)
    assert codes.codes_wrong(kind, c, c, zero.ctypes.data, 2) == 0


def test_logarithm_of_a_fraction(codes):
    """Against 40 digits.  Roundings: the table's entry and the series' last sum 2^-53
    of 2^-l each, their product 2^-53, the fma 2^-54, times log2(e): below 2^-50.6; the
    sum with l 2^-54.  The third term of the series of log2(1 + d), |d| < 2^-18.5: 2^-56."""
    ctx = decimal.Context(prec=40)
    ln2 = ctx.ln(decimal.Decimal(2))
    rng = np.random.default_rng(1)
    worst = 0.0
    fs = np.concatenate([1.0 + rng.random(300), 1.0 + 2.0 ** -rng.integers(1, 24, 40).astype(float),
                         2.0 - 2.0 ** -rng.integers(1, 24, 40).astype(float), [1.0]])
    for f in fs.astype(np.float32).astype(np.float64):
        if f >= 2.0:
            continue
        want = ctx.ln(decimal.Decimal(float(f))) / ln2
        for off in (0.0, 2.0 ** -20, -2.0 ** -20):
            worst = max(worst, abs(float(decimal.Decimal(codes.codes_log2(float(f), off)) - want)))
    assert worst <= 2.0 ** -50
