"""CPU tier: refusals at the ends of ranges (none reaches a device): grids of 2^32 threads,
which no launch takes, and numbers that are not fp32 values."""
import ctypes

import pytest

from cudaforge_amd import _lib

f = ctypes.c_float


@pytest.mark.parametrize("T", [(1 << 26) - 3, (1 << 26) - 1, 1 << 26, (1 << 31) - 1])
def test_gather(T):
    rc = _lib.load().cfa_kv_gather(256, 256, 256, 256, 0, 8, 2, 1, 2, 16, 64, 256, 4, 256, None, T,
                                   1, 256, 256, None)
    assert rc == _lib.CFA_ERR_ARG and "too many" in _lib.last_error()


@pytest.mark.parametrize("T", [(1 << 25) - 1, 1 << 25, (1 << 31) - 1])
def test_write(T):
    """One head of each kind: a wave for q, one for k and v."""
    rc = _lib.load().cfa_qk_norm_rope_kv_e4m3(
        256, 48, 16, 256, 48, 16, 256, 48, 16, 0, 256, T, 1, None, 1, 1, 16, 16, 256, f(1.0), 0, None,
        None, 0, f(1e-6), 256, 256, 256, 256, 256, 8, 2, 1, 16, 256, 4, 256, None)
    assert rc == _lib.CFA_ERR_ARG and "too many" in _lib.last_error()


@pytest.mark.parametrize("T", [(1 << 27) - 1, 1 << 27])
def test_merge(T):
    """Two splits of 16-bit pools, a merge's thread for four values."""
    lib = _lib.load()
    need = lib.cfa_prompt_attention_cached_workspace_size(T, 1, 1, 1, 128, T, 128, 0, 0, 0, 2)
    rc = lib.cfa_prompt_attention_cached(
        256, 256, 256, None, None, 0, 256, 1 << 20, 256, 8, 1, 0, 16, 256, T, 1, 1, 1, 128, f(0.1),
        f(0.0), None, 0, 0, T, 128, 2, 256, 256, need, None)
    assert rc == _lib.CFA_ERR_ARG and "too many" in _lib.last_error()


@pytest.mark.parametrize("r,fr,p", [(float("inf"), 0, 0), (1e39, 0, 0), (1e-50, 0, 0), (1, 1e39, 0),
                                    (1, float("nan"), 0), (1, 0, -1e39), (1, 0, float("inf"))])
def test_penalties(r, fr, p):
    rc = _lib.load().cfa_adjust_logits(256, 100, 100, 1, 2, 1, 100, 256, None, None, 5, None, f(r),
                                       None, f(fr), None, f(p), None, None, 0, None, None, 0, 0,
                                       None, 0, 0, None, 256, 100, 100, 0, None)
    assert rc == _lib.CFA_ERR_ARG
    assert "finite" in _lib.last_error()
