"""Rows of a cache in 8 bits, in plain 64-bit arithmetic: codes of 4 bits of
exponent and 3 of mantissa, with a power-of-two scale a row."""
import torch

TOP = 448.0


def values(codes, scales):
    """What codes [.., D] (any 8-bit type) and bytes [..] stand for, fp64, from the
    bits: (1 + m / 8) 2^(e - 7), below that steps of 2^-9; 0x7f is NaN."""
    c = codes.view(torch.uint8).long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (1 + m / 8) * torch.exp2(e.double() - 7), m * 2.0 ** -9)
    v = torch.where((c & 127) == 127, float("nan"), v)
    return torch.where(c >= 128, -v, v) * torch.exp2(scales.double() - 127)[..., None]


def scale_of(top):
    """The least power of two from 2^-126 on that brings top [..] to 448 or less."""
    e = torch.full(top.shape, -126.0, dtype=torch.float64)
    for _ in range(300):
        e = torch.where(top > TOP * torch.exp2(e), e + 1, e)
    return torch.exp2(e)


def step(y):
    """The distance of neighbouring codes at magnitude y (of a value over its scale)."""
    return torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)


def quantised(x):
    """(values, scales) of rows x [.., D] fp64, rounded to nearest even; what is not
    finite is NaN and does not count for the scale."""
    x = x.double()
    s = scale_of(torch.where(x.isfinite(), x.abs(), 0.0).amax(-1))
    y = torch.where(x.isfinite(), x, 0.0) / s[..., None]
    d = step(y)
    v = torch.round(y / d) * d * s[..., None]
    return torch.where(x.isfinite(), v, float("nan")), s


def random_pool(shape, g, spread=1.0):
    """Codes (float8_e4m3fn) and scales of a pool [.., D] of rows of different sizes."""
    size = torch.exp2(torch.randn(shape[:-1], generator=g) * spread)
    x = torch.randn(shape, generator=g) * size[..., None]
    s = scale_of(x.abs().amax(-1).double())
    codes = (x.double() / s[..., None]).float().to(torch.float8_e4m3fn)
    return codes, (torch.log2(s) + 127).to(torch.uint8)
