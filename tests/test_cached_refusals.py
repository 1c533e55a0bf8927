"""CPU tier: refusals of the entry points of the 8-bit cache and of adjust_logits
(none reaches a device) and their workspace sizes."""
import ctypes

import pytest
import torch

from cudaforge_amd import _lib
from cudaforge_amd.rotary import qk_norm_rope_kv
from cudaforge_amd.sampling import adjust_logits
from cudaforge_amd.verify import (kv_commit, kv_gather, prompt_attention,
                                  prompt_attention_workspace_bytes, tree_attention,
                                  tree_attention_workspace_bytes)

f = ctypes.c_float


def _refused(call, change, msg):
    assert call(**change) == _lib.CFA_ERR_ARG
    assert msg in _lib.last_error()


ATTENTION = dict(kp=256, vp=256, ks=256, vs=256, D=64, window=0, sinks=0, keys=64, splits=0, layer=0)


def _tree(**change):
    a = {**ATTENTION, **change}
    return _lib.load().cfa_tree_attention_cached(
        256, a["kp"], a["vp"], a["ks"], a["vs"], 0, 256, 8, 256, 8, 1, a["layer"], 16, 256, 0, 2,
        15, 0, 8, 2, a["D"], f(0.1), f(0.0), None, a["window"], a["sinks"], a["keys"], a["splits"],
        256, None, 0, None)


def _prompt(**change):
    a = {**ATTENTION, **change}
    return _lib.load().cfa_prompt_attention_cached(
        256, a["kp"], a["vp"], a["ks"], a["vs"], 0, 256, 8, 256, 8, 1, a["layer"], 16, 256, 30, 2,
        8, 2, a["D"], f(0.1), f(0.0), None, a["window"], a["sinks"], 20, a["keys"], a["splits"],
        256, None, 0, None)


@pytest.mark.parametrize("call", [_tree, _prompt])
@pytest.mark.parametrize("change,msg", [
    (dict(ks=None), "go together"), (dict(vs=None), "go together"), (dict(ks=264), "aligned"),
    (dict(vs=257), "aligned"), (dict(kp=264), "aligned"), (dict(sinks=-1), "sinks"),
    (dict(window=-1), "window"), (dict(D=80), "head_dim"), (dict(layer=1), "geometry"),
    (dict(splits=2, keys=128), "workspace")])
def test_attention(call, change, msg):
    _refused(call, change, msg)


def test_attention_workspaces():
    # 4 splits x 2 x 15 x 8 rows: fp32 sums of 64, then (base, sum); the cache's type
    # and the first tokens change the plan, not what a split leaves
    want = 4 * 2 * 15 * 8 * (64 + 2) * 4
    for e4m3 in (False, True):
        got = tree_attention_workspace_bytes(2, 15, 8, 2, 64, 1000, 4, scored=True, window=300,
                                             sinks=64, e4m3=e4m3)
        assert got == want
        assert tree_attention_workspace_bytes(2, 15, 8, 2, 64, 60, 1, scored=True, e4m3=e4m3) == 0
        assert prompt_attention_workspace_bytes(30, 2, 8, 2, 64, 15, 1000, num_splits=4,
                                                e4m3=e4m3) == want


GATHER = dict(kp=256, vp=256, ks=256, vs=256, nblk=8, layers=2, layer=1, Hkv=2, bs=16, D=64,
              maxb=4, starts=256, T=6, B=2, ko=256, vo=256)


def _gather(**change):
    a = {**GATHER, **change}
    return _lib.load().cfa_kv_gather(
        a["kp"], a["vp"], a["ks"], a["vs"], 0, a["nblk"], a["layers"], a["layer"], a["Hkv"], a["bs"],
        a["D"], 256, a["maxb"], a["starts"], None, a["T"], a["B"], a["ko"], a["vo"], None)


@pytest.mark.parametrize("change,msg", [
    (dict(T=-1), "T, B >= 0"), (dict(B=-1), "T, B >= 0"), (dict(Hkv=0), "heads"),
    (dict(D=72), "multiple of 16"), (dict(D=272), "at most 256"), (dict(D=0), "head_dim"),
    (dict(nblk=0), "geometry"), (dict(layer=2), "geometry"), (dict(layer=-1), "geometry"),
    (dict(bs=0), "geometry"), (dict(maxb=-1), "geometry"), (dict(ks=None), "go together"),
    (dict(kp=None), "null"), (dict(starts=None), "null"), (dict(vo=None), "null"),
    (dict(T=5), "multiple of B"), (dict(ko=258), "aligned"), (dict(vp=264), "aligned"),
    (dict(T=1 << 26), "too many")])
def test_gather(change, msg):
    _refused(_gather, change, msg)


def test_gather_of_nothing():
    assert _gather(T=0, ko=None, vo=None, kp=None) == _lib.CFA_OK
    assert _gather(B=0, ko=None, starts=None) == _lib.CFA_OK


def _commit(**change):
    a = {**dict(ks=256, vs=256, D=64), **change}
    return _lib.load().cfa_kv_commit_scaled(256, 256, a["ks"], a["vs"], 256, 4, 256, 256, 7, 256, 2,
                                            8, 1, 2, 16, a["D"], 1, 256, 256, None)


@pytest.mark.parametrize("change,msg", [(dict(ks=None), "go together"),
                                        (dict(vs=None), "go together"), (dict(D=24), "16")])
def test_commit(change, msg):
    _refused(_commit, change, msg)


def _write(**change):
    a = {**dict(kp=256, vp=256, ks=256, vs=256, D=64, rot=64, layer=1), **change}
    return _lib.load().cfa_qk_norm_rope_kv_e4m3(
        256, 256, 64, 256, 128, 64, 256, 128, 64, 0, 256, 6, 2, None, 4, 2, a["D"], a["rot"], 256,
        f(1.0), 0, None, None, 0, f(1e-6), 256, a["kp"], a["vp"], a["ks"], a["vs"], 8, 2, a["layer"],
        16, 256, 4, 256, None)


@pytest.mark.parametrize("change,msg", [
    (dict(ks=None), "go together"), (dict(vs=None), "go together"), (dict(D=72), "multiple of 16"),
    (dict(kp=264), "aligned"), (dict(vp=257), "aligned"), (dict(rot=66), "rotary_dim"),
    (dict(layer=2), "geometry")])
def test_write(change, msg):
    _refused(_write, change, msg)


LOGITS = dict(x=256, type=1, B=2, N=3, V=100, history=256, L=5, r=1.0, nodes=None, mask=None, bt=256,
              bv=256, K=2, allowed=256, words=4, masks=6, out=256)


def _adjust(**change):
    a = {**LOGITS, **change}
    return _lib.load().cfa_adjust_logits(
        a["x"], 300, 100, a["type"], a["B"], a["N"], a["V"], a["history"], None, None, a["L"], None,
        f(a["r"]), None, f(0.0), None, f(0.0), a["nodes"], a["mask"], 0, a["bt"], a["bv"], 0, a["K"],
        a["allowed"], a["words"], a["masks"], None, a["out"], 300, 100, 0, None)


@pytest.mark.parametrize("change,msg", [
    (dict(B=-1), "B, N, L, K"), (dict(N=-1), "B, N, L, K"), (dict(V=0), "V > 0"),
    (dict(L=-1), "B, N, L, K"), (dict(K=-1), "B, N, L, K"), (dict(type=3), "type"),
    (dict(type=-1), "type"), (dict(N=65, nodes=256, mask=256), "64"), (dict(nodes=256), "together"),
    (dict(mask=256), "together"), (dict(r=0.0), "positive"), (dict(r=float("nan")), "positive"),
    (dict(words=3), "bit for every token"), (dict(masks=-1), "bit for every token"),
    (dict(x=None), "null"), (dict(out=None), "null"), (dict(history=None), "null"),
    (dict(bv=None), "null"), (dict(B=2 ** 22, N=1), "too many")])
def test_adjust(change, msg):
    _refused(_adjust, change, msg)


def test_adjusting_nothing():
    assert _adjust(B=0, x=None, out=None) == _lib.CFA_OK
    assert _adjust(N=0, x=None, out=None) == _lib.CFA_OK


def test_host_tensors_are_refused():
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 1, 4, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros(2, 1, 4, 16, dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    t, scales = i.view(2, 1), dict(k_scales=s, v_scales=s)
    for call in (lambda: kv_gather(pool, pool, t, i, tokens=2, **scales),
                 lambda: kv_commit(pool, pool, t, i, t, i, **scales),
                 lambda: qk_norm_rope_kv(q, q, q, i, None, pool, pool, t, i, **scales),
                 lambda: tree_attention(q[:, None], pool, pool, t, i, i.long()[:1], **scales),
                 lambda: prompt_attention(q, pool, pool, t, i, i, **scales),
                 lambda: adjust_logits(torch.zeros(2, 9))):
        with pytest.raises(ValueError, match="device tensor"):
            call()
