"""CPU tier: refusals of cfa_sample_rows and sample_rows (no device reached)."""
import ctypes

import pytest
import torch

from cudaforge_amd import _lib
from cudaforge_amd.sampling import filtered_probs, sample_rows, sample_rows_workspace_bytes

GOOD = dict(rows=256, stride=1000, type=0, R=4, V=1000, draws=1, u=256, tok=256, probs=None, ws=256,
            wsn=1 << 30)


def _call(**change):
    a = {**GOOD, **change}
    f = ctypes.c_float
    return _lib.load().cfa_sample_rows(
        a["rows"], a["stride"], a["type"], a["R"], a["V"], a["draws"], None, f(1.0), None, 0, None,
        f(1.0), None, f(0.0), a["u"], a["tok"], a["probs"], a["ws"], a["wsn"], None)


@pytest.mark.parametrize("change,msg", [
    (dict(R=-1), "R >= 0"), (dict(V=0), "V <= 2^20"), (dict(V=2 ** 20 + 1, stride=2 ** 21), "V <= 2^20"),
    (dict(type=3), "elem_type"), (dict(type=-1), "elem_type"), (dict(draws=-1), "draws"),
    (dict(draws=65), "draws"), (dict(draws=0), "out_probs"), (dict(stride=999), "row_stride"),
    (dict(rows=None), "null"), (dict(u=None), "null"), (dict(tok=None), "null"), (dict(ws=None), "null"),
    (dict(wsn=100), "workspace"), (dict(ws=257), "aligned"), (dict(probs=257), "aligned"),
    (dict(R=2 ** 24), "workspace"), (dict(R=2 ** 23, wsn=1 << 40), "too many")])
def test_entry_point_refusals(change, msg):
    assert _call(**change) == _lib.CFA_ERR_ARG
    assert msg in _lib.last_error()


def test_nothing_to_draw_launches_nothing():
    assert _call(R=0, rows=None, ws=None) == _lib.CFA_OK


def test_workspace_size():
    # per 8192 tokens: the maximum and 512 bins; per row its cut
    def up(x):
        return -(-x // 256) * 256

    for R, V in ((1, 1), (3, 8192), (64, 128256), (2, 2 ** 20)):
        n = R * -(-V // 8192)
        assert sample_rows_workspace_bytes(R, V) == up(4 * n) + up(n * 4096) + up(32 * R)
    assert sample_rows_workspace_bytes(0, 10) == 0
    assert sample_rows_workspace_bytes(1, 2 ** 20 + 1) == 0


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="device tensor"):
        sample_rows(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="device tensor"):
        filtered_probs(torch.zeros(2, 8))
