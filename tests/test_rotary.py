"""CPU tier: frequencies of rotary.Rotary against their formulas, and the
refusals of qk_norm_rope_kv and its C entry point, none of which reach a
device."""
import ctypes
import math

import numpy as np
import pytest
import torch

from cudaforge_amd import _lib
from cudaforge_amd.rotary import Rotary, qk_norm_rope_kv


def _radians(r):
    bits = r.turns.numpy().view(np.uint64)
    return np.array([int(b) for b in bits], dtype=object) * (2 * math.pi) / 2.0 ** 64


@pytest.mark.parametrize("rot,theta", [(128, 10000.0), (64, 500000.0), (2, 10000.0), (0, 10000.0)])
def test_plain_frequencies(rot, theta):
    r = Rotary(rot, theta)
    want = [theta ** (-2 * i / rot) for i in range(rot // 2)]
    np.testing.assert_allclose(r.radians.numpy(), want, rtol=1e-15)
    # the fixed-point turn: off by its own last place and fp64's rounding
    np.testing.assert_allclose(_radians(r).astype(float), want, rtol=4e-16, atol=2.0 ** -61)
    assert r.factor == 1.0 and r.rotary_dim == rot


def test_scalings():
    rot, theta = 128, 500000.0
    inv = np.array([theta ** (-2 * i / rot) for i in range(64)])
    lin = Rotary(rot, theta, scaling=dict(kind="linear", factor=4.0))
    np.testing.assert_allclose(lin.radians.numpy(), inv / 4.0, rtol=1e-15)
    ntk = Rotary(rot, theta, scaling=dict(kind="ntk", factor=4.0))
    t2 = theta * 4.0 ** (rot / (rot - 2))
    np.testing.assert_allclose(ntk.radians.numpy(), [t2 ** (-2 * i / rot) for i in range(64)],
                               rtol=1e-14)
    # bands: pairs by the wavelength they have
    b = Rotary(rot, theta, scaling=dict(kind="bands", factor=8.0, low=1.0, high=4.0,
                                        original=8192)).radians.numpy()
    for i in range(64):
        wave = 2 * math.pi / inv[i]
        if wave < 8192 / 4.0:
            want = inv[i]
        elif wave > 8192 / 1.0:
            want = inv[i] / 8.0
        else:
            s = (8192 / wave - 1.0) / 3.0
            want = (1 - s) * inv[i] / 8.0 + s * inv[i]
        assert abs(b[i] - want) <= 1e-14 * want
    y = Rotary(rot, theta, scaling=dict(kind="yarn", factor=16.0, original=4096))
    assert abs(y.factor - (0.1 * math.log(16.0) + 1.0)) < 1e-15
    assert y.radians[0] == inv[0]
    np.testing.assert_allclose(y.radians.numpy()[-1], inv[-1] / 16.0, rtol=1e-14)
    ratio = y.radians.numpy() / inv
    assert (np.diff(ratio) <= 1e-15).all()
    assert Rotary(rot, theta, scaling=dict(kind="yarn", factor=16.0, original=4096,
                                           attention_factor=1.0)).factor == 1.0


def test_from_frequencies_takes_whole_turns_away():
    a = Rotary.from_frequencies([0.25, 0.5])
    b = Rotary.from_frequencies([0.25 + 2 * math.pi, 0.5 + 4 * math.pi], layout="interleaved")
    d = (a.turns - b.turns).numpy().astype(float) / 2.0 ** 64
    assert np.abs(d).max() < 1e-15
    assert b.layout == "interleaved"


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=7), dict(rotary_dim=-2), dict(rotary_dim=8, layout="other"),
    dict(rotary_dim=8, theta=0.0), dict(rotary_dim=8, theta=float("nan")),
    dict(rotary_dim=8, scaling=dict(kind="other")),
    dict(rotary_dim=8, scaling=dict(kind="linear")),
    dict(rotary_dim=8, scaling=dict(kind="linear", factor=0.0)),
    dict(rotary_dim=8, scaling=dict(kind="linear", factor=2.0, low=1.0)),
    dict(rotary_dim=2, scaling=dict(kind="ntk", factor=2.0)),
    dict(rotary_dim=8, scaling=dict(kind="bands", factor=2.0, low=4.0, high=1.0, original=64)),
    dict(rotary_dim=8, scaling=dict(kind="yarn", factor=2.0)),
])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        Rotary(**kw)
    with pytest.raises(ValueError):
        Rotary.from_frequencies([float("inf")])


def test_host_tensors_are_refused():
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 1, 4, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        qk_norm_rope_kv(q, q, q, i, None, pool, pool, i.view(2, 1), i)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        qk_norm_rope_kv(q.float(), q, q, i, None, pool, pool, i.view(2, 1), i)


GOOD = dict(T=6, B=2, Hq=4, Hkv=2, D=64, rot=64, nblk=8, layers=2, layer=1, bs=16, maxb=4)


@pytest.mark.parametrize("change,msg", [
    (dict(T=-1), "T, B >= 0"), (dict(B=-1), "T, B >= 0"), (dict(Hq=0), "head counts"),
    (dict(Hkv=0), "head counts"), (dict(D=60, rot=0), "head_dim"), (dict(D=264), "head_dim"),
    (dict(rot=66), "rotary_dim"), (dict(rot=7), "rotary_dim"), (dict(rot=-2), "rotary_dim"),
    (dict(nblk=0), "geometry"), (dict(layer=2), "geometry"), (dict(layer=-1), "geometry"),
    (dict(bs=0), "geometry"), (dict(maxb=-1), "geometry"), (dict(T=5), "multiple of B"),
    (dict(null="q"), "null"), (dict(null="turns"), "null"), (dict(null="base"), "null"),
    (dict(T=2 ** 26), "too many"),
])
def test_entry_point_refusals(change, msg):
    """Shape checks run before anything touches a device (dummy pointers)."""
    a = {**GOOD, **change}
    p = {n: (None if a.get("null") == n else 256) for n in ("q", "turns", "base")}
    rc = _lib.load().cfa_qk_norm_rope_kv(
        p["q"], 256, 64, 256, 128, 64, 256, 128, 64, 0, 256, a["T"], a["B"], None, a["Hq"],
        a["Hkv"], a["D"], a["rot"], p["turns"], ctypes.c_float(1.0), 0, None, None, 0,
        ctypes.c_float(1e-6), 256, 256, 256, a["nblk"], a["layers"], a["layer"], a["bs"], 256,
        a["maxb"], p["base"], None)
    assert rc == _lib.CFA_ERR_ARG
    assert msg in _lib.last_error()


@pytest.mark.parametrize("change", [dict(T=0), dict(B=0, T=0), dict(T=4, B=0)])
def test_nothing_to_do_launches_nothing(change):
    a = {**GOOD, **change}
    rc = _lib.load().cfa_qk_norm_rope_kv(
        None, 256, 64, None, 128, 64, None, 128, 64, 0, None, a["T"], a["B"], None, a["Hq"],
        a["Hkv"], a["D"], a["rot"], None, ctypes.c_float(1.0), 0, None, None, 0,
        ctypes.c_float(1e-6), None, None, None, a["nblk"], a["layers"], a["layer"], a["bs"], None,
        a["maxb"], None, None)
    assert rc == _lib.CFA_OK


@pytest.mark.parametrize("scaling", [dict(kind="linear", factor=None), dict(kind="ntk", factor=None),
                                     dict(kind="bands", factor=8.0, low=None, high=4.0, original=8192),
                                     dict(kind="yarn", factor=None, original=4096)])
def test_a_scaling_without_its_value_is_refused(scaling):
    """None is no value: it is not taken for a factor of 1."""
    with pytest.raises(ValueError, match="missing"):
        Rotary(64, scaling=scaling)


def test_optional_scaling_values_may_be_none():
    a = Rotary(64, scaling=dict(kind="yarn", factor=4.0, original=4096, fast=None,
                                attention_factor=None))
    b = Rotary(64, scaling=dict(kind="yarn", factor=4.0, original=4096))
    assert torch.equal(a.turns, b.turns) and a.factor == b.factor
