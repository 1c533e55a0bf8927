"""GPU tier: the codes of written keys are their exact values', rounded once, whatever
the weights' type; and every form of the launch writes the same bits."""
import math

import pytest
import torch

from cudaforge_amd.rotary import Rotary, qk_norm_rope_kv
from tests import e4m3_reference as E

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
F8 = torch.float8_e4m3fn


def _exponent(x):
    """floor(log2 x) of x > 0, fp64."""
    return torch.frexp(x)[1].double() - 1


def _exact(x, w, pos, rotary, eps):
    """Keys x [T, H, D] in 64 bits and the magnitudes that went into them."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    r = rotary.rotary_dim
    # the angle in turns: integers modulo 2^64
    turn = (pos.long()[:, None] * rotary.turns[None]).double() * 2.0 ** -64
    cos = (2 * math.pi * turn).cos()[:, None] * rotary.factor
    sin = (2 * math.pi * turn).sin()[:, None] * rotary.factor
    i = torch.arange(r // 2, device=x.device)
    ia, ib = (i, i + r // 2) if rotary.layout == "half" else (2 * i, 2 * i + 1)
    a, b = y[..., ia], y[..., ib]
    mag = y.abs()
    y = y.clone()
    y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * rotary.factor
    return y, mag


def _write(x, w, pos, rotary, Hkv, dtype, eps=1e-6):
    """The keys' values (fp64, by their codes) and scales' exponents, [T, Hkv]."""
    T, D = x.shape[0], x.shape[2]
    pages = (T + 15) // 16
    pools = [torch.zeros(pages, 1, Hkv, 16, D, dtype=torch.uint8, device=x.device).view(F8)
             for _ in range(2)]
    scales = [torch.zeros(pages, 1, Hkv, 16, dtype=torch.uint8, device=x.device) for _ in range(2)]
    qk_norm_rope_kv(x[:, :1], x[:, 1:], x[:, 1:], pos, rotary, *pools,
                    torch.arange(pages, dtype=torch.int32, device=x.device)[None],
                    torch.zeros(1, dtype=torch.int32, device=x.device), k_norm=w, eps=eps,
                    k_scales=scales[0], v_scales=scales[1])
    got = E.values(pools[0], scales[0])[:, 0].transpose(1, 2).reshape(-1, Hkv, D)[:T]
    return got, scales[0][:, 0].transpose(1, 2).reshape(-1, Hkv)[:T].double() - 127


def _check_codes(got, e, want, mag):
    """Within half a code's step of the exact value, but for what the arithmetic in 64 bits
    is off by: the polynomials of sine and cosine (2^-34 and 2^-37 of theirs), the root's
    one step of Newton's (2^-43) and some roundings of 2^-53, less than 2^-32 (|a| + |b|)
    in all.  The largest of a row sets its scale: 448 2^e is not below it."""
    tol = 2.0 ** -32 * mag
    top, at = want.abs().max(-1)
    off = tol.gather(-1, at[..., None])[..., 0]
    least = [torch.where(m > E.TOP * torch.exp2(_exponent(m) - 8), _exponent(m) - 7,
                         _exponent(m) - 8) for m in (top - off, top + off)]
    assert ((e == least[0]) | (e == least[1])).all()
    y = (want.abs() + tol) * torch.exp2(-e)[..., None]
    half = torch.exp2(_exponent(y.clamp(min=2.0 ** -6)) - 4 + e[..., None])
    bad = (got - want).abs() > half + tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}"


@pytest.mark.parametrize("dtype,norm,layout", [(BF, BF, "half"), (BF, F32, "half"),
                                               (HF, F32, "interleaved"), (HF, HF, "half"),
                                               (BF, None, "interleaved")])
def test_codes_of_keys(device, dtype, norm, layout):
    """16 million keys' codes."""
    g = torch.Generator(device=device).manual_seed(3)
    T, Hkv, D = 8000, 16, 128
    x = torch.randn(T, 1 + Hkv, D, generator=g, device=device).to(dtype)
    w = None if norm is None else (1 + 0.3 * torch.randn(D, generator=g, device=device)).to(norm)
    pos = torch.randint(-200000, 200000, (T,), generator=g, device=device, dtype=torch.int32)
    rotary = Rotary(D, 500000.0, layout=layout, device=device)
    got, e = _write(x, w, pos, rotary, Hkv, dtype)
    _check_codes(got, e, *_exact(x[:, 1:], w, pos, rotary, 1e-6))


@pytest.mark.parametrize("D,rot,layout", [(64, 64, "half"), (128, 64, "interleaved"), (80, 40, "half"),
                                          (256, 256, "half"), (32, 20, "half")])
def test_weights_of_32_bits(device, D, rot, layout):
    """Parts of heads, and pairs whose weights differ by far."""
    g = torch.Generator(device=device).manual_seed(4)
    T, Hkv = 900, 4
    x = torch.randn(T, 1 + Hkv, D, generator=g, device=device).to(BF)
    w = torch.exp2(3 * torch.randn(D, generator=g, device=device))
    pos = torch.randint(0, 200000, (T,), generator=g, device=device, dtype=torch.int32)
    rotary = Rotary(rot, 10000.0, layout=layout, device=device)
    got, e = _write(x, w, pos, rotary, Hkv, BF)
    _check_codes(got, e, *_exact(x[:, 1:], w, pos, rotary, 1e-6))


@pytest.mark.parametrize("size,weight", [(1e10, 1e30), (1e25, 1.0), (1e37, 100.0), (1e-30, 1.0)])
def test_products_outside_the_range_of_fp32(device, size, weight):
    """The squares, or the products with the weights, are not fp32 values; the keys are."""
    g = torch.Generator(device=device).manual_seed(5)
    T, Hkv, D = 40, 2, 64
    x = (torch.randn(T, 1 + Hkv, D, generator=g, device=device) * size).to(BF)
    w = weight * (1 + 0.1 * torch.randn(D, generator=g, device=device))
    pos = torch.randint(0, 2000, (T,), generator=g, device=device, dtype=torch.int32)
    rotary = Rotary(D, 10000.0, device=device)
    got, e = _write(x, w, pos, rotary, Hkv, BF, eps=0.0)
    _check_codes(got, e, *_exact(x[:, 1:], w, pos, rotary, 0.0))


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,layout", [
    (700, 32, 8, 128, 128, "half"), (2800, 32, 8, 128, 128, "half"),
    (2000, 32, 8, 128, 64, "interleaved"), (3000, 20, 11, 128, 128, "half"),
    (3300, 33, 20, 64, 64, "interleaved"), (3300, 9, 5, 256, 256, "half"),
    (3000, 20, 11, 80, 40, "half"), (5000, 70, 17, 16, 16, "half"), (9000, 5, 3, 128, 0, "half")])
@pytest.mark.parametrize("dtype,norm", [(BF, F32), (HF, HF)])
def test_forms_of_the_launch(device, T, Hq, Hkv, D, rot, layout, dtype, norm):
    """Many tokens in one call, ragged, padded and with an unmapped page, whose waves take
    several rows and rounds of them, against the same tokens in calls of up to 100."""
    g = torch.Generator().manual_seed(6)
    first = T // 3
    lens = [first, 1, 0, T - first - 1]
    base = [5, 16, 3, 40]
    need = [(b + n + 15) // 16 for b, n in zip(base, lens)]
    perm = torch.randperm(sum(need), generator=g).int()
    bt = torch.full((4, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[at: at + n]
        at += n
    bt[3, 7] = -1
    x = torch.randn(T + 3, Hq + 2 * Hkv, D, generator=g).to(dtype).to(device)
    pos = torch.randint(0, 200000, (T + 3,), generator=g, dtype=torch.int32).to(device)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(norm).to(device) for _ in range(2))
    rotary = Rotary(rot, 500000.0, layout=layout, device=device) if rot else None
    bt = bt.to(device)
    q, k, v = x.split([Hq, Hkv, Hkv], 1)

    def pools():
        return ([torch.full((len(perm), 2, Hkv, 16, D), 1, dtype=torch.uint8, device=device).view(F8)
                 for _ in range(2)],
                [torch.full((len(perm), 2, Hkv, 16), 2, dtype=torch.uint8, device=device)
                 for _ in range(2)], torch.full_like(q, 5.0).contiguous())

    def write(to, rows, tables, lens, cu=None):
        codes, scales, out = to
        qk_norm_rope_kv(q[rows], k[rows], v[rows], pos[rows], rotary, *codes, tables,
                        torch.tensor(lens, dtype=torch.int32, device=device), layer=1,
                        cu_seqlens=cu, q_norm=wq, k_norm=wk, q_out=out[rows], k_scales=scales[0],
                        v_scales=scales[1])

    many, few = pools(), pools()
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)
    write(many, slice(0, T + 3), bt, base, cu.to(device))
    for b, n in enumerate(lens):
        for i in range(0, n, 100):
            t = int(cu[b]) + i
            write(few, slice(t, t + min(100, n - i)), bt[b: b + 1], [base[b] + i])
    for a, b in zip(many[0] + many[1], few[0] + few[1]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(many[2].view(torch.int16), few[2].view(torch.int16))
