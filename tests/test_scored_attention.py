"""CPU tier: refusals of the scored attention entry points (none reaches a
device) and their workspace sizes."""
import ctypes

import pytest
import torch

from cudaforge_amd import _lib
from cudaforge_amd.verify import (prompt_attention, prompt_attention_workspace_bytes, tree_attention,
                                  tree_attention_workspace_bytes)

TREE = dict(nblk=8, layers=1, layer=0, bs=16, maxb=8, B=2, N=15, first=0, Hq=8, Hkv=2, D=64,
            scale=0.1, cap=0.0, window=0, keys=64, splits=0, q=256, out=256)


def _tree(**change):
    a = {**TREE, **change}
    f = ctypes.c_float
    return _lib.load().cfa_tree_attention_scored(
        a["q"], 256, 256, 0, 256, a["maxb"], 256, a["nblk"], a["layers"], a["layer"], a["bs"], 256, 0,
        a["B"], a["N"], a["first"], a["Hq"], a["Hkv"], a["D"], f(a["scale"]), f(a["cap"]), None,
        a["window"], a["keys"], a["splits"], a["out"], None, 0, None)


COMMON = [(dict(Hq=0), "n_q_heads"), (dict(Hkv=3), "multiple"), (dict(Hq=514), "at most 256"),
          (dict(D=96), "head_dim"), (dict(bs=8), "block_size"), (dict(bs=0), "block_size"),
          (dict(nblk=0), "geometry"), (dict(layer=1), "geometry"), (dict(maxb=0), "max_blocks"),
          (dict(maxb=2 ** 30), "2\\^31"), (dict(scale=float("inf")), "sm_scale"),
          (dict(cap=-1.0), "soft_cap"), (dict(cap=float("nan")), "soft_cap"),
          (dict(cap=1e-7), "soft_cap"), (dict(window=-1), "window"), (dict(splits=-1), "num_splits")]


@pytest.mark.parametrize("change,msg", COMMON + [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(q=264), "aligned"),
    (dict(out=258), "aligned"), (dict(B=0), "B > 0"), (dict(N=65), "64"),
    (dict(N=0), "64"), (dict(first=15), "first_node"), (dict(first=-1), "first_node"),
    (dict(keys=14), "max_keys"), (dict(keys=129), "cover"), (dict(splits=2, keys=128), "workspace")])
def test_tree_refusals(change, msg):
    import re

    assert _tree(**change) == _lib.CFA_ERR_ARG
    assert re.search(msg, _lib.last_error())


def _prompt(**change):
    a = {**TREE, "T": 30, "mq": 20, **change}
    f = ctypes.c_float
    return _lib.load().cfa_prompt_attention(
        a["q"], 256, 256, 0, 256, a["maxb"], 256, a["nblk"], a["layers"], a["layer"], a["bs"], 256,
        a["T"], a["B"], a["Hq"], a["Hkv"], a["D"], f(a["scale"]), f(a["cap"]), None, a["window"],
        a["mq"], a["keys"], a["splits"], a["out"], None, 0, None)


@pytest.mark.parametrize("change,msg", COMMON + [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(q=264), "aligned"),
    (dict(out=258), "aligned"), (dict(T=-1), "T, B"), (dict(B=-1), "T, B"),
    (dict(mq=0), "max_query"), (dict(keys=0), "max_keys"), (dict(splits=2, keys=128), "workspace"),
    (dict(T=2 ** 30), "too many")])
def test_prompt_refusals(change, msg):
    import re

    assert _prompt(**change) == _lib.CFA_ERR_ARG
    assert re.search(msg, _lib.last_error())


def test_empty_prompts_launch_nothing():
    assert _prompt(T=0, q=None, out=None) == _lib.CFA_OK
    assert _prompt(B=0, q=None, out=None) == _lib.CFA_OK


def test_workspace_sizes():
    # 4 splits x 2 x 15 x 8 rows: fp32 sums of 64, then (base, sum)
    rows = 4 * 2 * 15 * 8
    want = rows * 64 * 4 + rows * 8
    assert tree_attention_workspace_bytes(2, 15, 8, 2, 64, 1000, 4, scored=True) == want
    # a window of 100 spans few tiles, whatever the context
    assert tree_attention_workspace_bytes(2, 15, 8, 2, 64, 10 ** 6, 50, window=100) \
        == 4 * (2 * 15 * 8) * (64 * 4 + 8)
    assert tree_attention_workspace_bytes(2, 15, 8, 2, 64, 1000, 1, scored=True) == 0
    assert prompt_attention_workspace_bytes(30, 2, 8, 2, 64, 20, 1000, 0, 4) \
        == -(-4 * 30 * 8 * 64 * 4 // 256) * 256 + -(-4 * 30 * 8 * 8 // 256) * 256
    # enough blocks to fill the device need none
    assert prompt_attention_workspace_bytes(8192, 1, 32, 8, 128, 8192, 8192) == 0
    lib = _lib.load()
    assert lib.cfa_prompt_attention_workspace_size(30, 2, 8, 3, 64, 20, 1000, 0, 4) == 0
    assert lib.cfa_tree_attention_scored_workspace_size(0, 15, 8, 2, 64, 1000, 0, 4) == 0


def test_host_tensors_are_refused():
    q = torch.zeros(1, 3, 8, 64, dtype=torch.bfloat16)
    pool = torch.zeros(4, 1, 2, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        tree_attention(q, pool, pool, i.view(1, 1), i, torch.ones(3, dtype=torch.int64), soft_cap=50.0)
    with pytest.raises(ValueError, match="device tensor"):
        prompt_attention(q[0], pool, pool, i.view(1, 1), i, torch.zeros(2, dtype=torch.int32))


def test_workspace_elsewhere_is_refused():
    """Before a device is reached: its address is the host's."""
    from cudaforge_amd.verify import _workspace

    there = torch.device("cuda", 0)
    for n in (4, 4096):
        with pytest.raises(ValueError, match="workspace"):
            _workspace(torch.empty(n, dtype=torch.uint8), 64, there)
    with pytest.raises(TypeError, match="workspace"):
        _workspace([0] * 64, 64, there)


def test_scales_past_fp32_are_refused():
    for call in (_tree, _prompt):
        for change in (dict(scale=3e38), dict(scale=-3e38), dict(scale=1e33, cap=1e-6),
                       dict(scale=1.2e38, cap=1.0)):
            assert call(**change) == _lib.CFA_ERR_ARG
            assert "sm_scale" in _lib.last_error()
        # (refused for something else, behind the scale's check)
        assert call(scale=2e38, keys=0) == _lib.CFA_ERR_ARG and "max_keys" in _lib.last_error()


def test_bounds_past_32_bits():
    far, most = 2 ** 32 + 5, 2 ** 31 - 1
    for w, k in ((far, 1000), (0, far), (far, far)):
        assert tree_attention_workspace_bytes(2, 15, 8, 2, 64, k, 4, scored=True, window=w) \
            == tree_attention_workspace_bytes(2, 15, 8, 2, 64, min(k, most), 4, scored=True,
                                              window=min(w, most)) > 0
        assert prompt_attention_workspace_bytes(30, 2, 8, 2, 64, far, k, w, 4) \
            == prompt_attention_workspace_bytes(30, 2, 8, 2, 64, most, min(k, most), min(w, most), 4) > 0
