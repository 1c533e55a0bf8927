"""Rotary positions, with RMSNorm of the q and k heads and the paged-cache
write in the same pass (``cfa_qk_norm_rope_kv``).

The reference has the half-split rotation of whole heads alone
(``csrc/include/cudaforge/kernels/rope.cuh:35-66``).  ``Rotary`` holds a
model's frequencies: either layout (halves or neighbours), part of a head,
and the usual scalings for contexts longer than the trained one.
``qk_norm_rope_kv`` applies them to a QKV projection and fills the pages that
``verify.tree_attention`` and ``verify.prompt_attention`` read.
"""
from __future__ import annotations

import math
from typing import Optional

import numpy as np
import torch

from . import _lib
from .verify import _on, _ptr, _require_all, _require_cuda, _stream_ptr

__all__ = ["Rotary", "qk_norm_rope_kv"]

_LAYOUTS = ("half", "interleaved")


class Rotary:
    """Frequencies of a rotary embedding, on the device.

    ``rotary_dim`` elements of each head (the first ones) turn in pairs:
    ``layout`` "half" pairs (i, i + rotary_dim / 2), "interleaved" (2i, 2i + 1).
    Pair i turns by ``theta ** (-2 i / rotary_dim)`` radians per position,
    changed by ``scaling`` (a dict, None: as they are):

      kind "linear"  every frequency / factor
      kind "ntk"     theta * factor ** (rotary_dim / (rotary_dim - 2))
      kind "bands"   by the turns a pair makes over `original` positions: at
                     least `high` keeps its frequency, at most `low` has it
                     divided by factor, linear in the turns between
      kind "yarn"    a ramp over the pairs from the one that makes `fast` turns
                     over `original` positions (default 32, kept) to the one
                     that makes `slow` (default 1, divided by factor), and q and
                     k multiplied by `attention_factor` (default
                     0.1 ln(factor) + 1)

    The frequencies are kept as 64-bit fractions of a turn (``turns``, int64
    bits), so an angle is exact modulo a turn at every 32-bit position.
    """

    def __init__(self, rotary_dim: int, theta: float = 10000.0, *, layout: str = "half",
                 scaling: Optional[dict] = None, device=None):
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {_LAYOUTS}")
        if rotary_dim < 0 or rotary_dim % 2:
            raise ValueError("rotary_dim must be even and not negative")
        if not theta > 0.0 or not math.isfinite(theta):
            raise ValueError("theta must be positive and finite")
        inv, factor = self._frequencies(int(rotary_dim), float(theta), dict(scaling or {}))
        self._set(inv, layout, factor, device)

    @classmethod
    def from_frequencies(cls, radians, *, layout: str = "half", factor: float = 1.0, device=None
                         ) -> "Rotary":
        """From each pair's radians per position (any sequence of floats);
        ``factor`` multiplies the turned q and k."""
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {_LAYOUTS}")
        r = cls.__new__(cls)
        r._set(np.asarray(radians, dtype=np.float64).reshape(-1), layout, float(factor), device)
        return r

    def _set(self, inv: np.ndarray, layout: str, factor: float, device) -> None:
        if not np.isfinite(inv).all() or not math.isfinite(factor):
            raise ValueError("frequencies must be finite")
        self.rotary_dim = 2 * len(inv)
        self.layout = layout
        self.factor = factor
        self.radians = torch.from_numpy(inv.copy())
        # a scaling by 2^64 is exact; whole turns fall away
        bits = [int(math.ldexp(f / (2.0 * math.pi), 64)) & (2 ** 64 - 1) for f in inv]
        self.turns = torch.from_numpy(np.array(bits, dtype=np.uint64).view(np.int64))
        if device is not None:
            self.turns = self.turns.to(device)

    @staticmethod
    def _frequencies(r: int, theta: float, sc: dict):
        kind = sc.pop("kind", None)
        takes = {None: (), "linear": ("factor",), "ntk": ("factor",),
                 "bands": ("factor", "low", "high", "original"),
                 "yarn": ("factor", "original")}
        if kind not in takes:
            raise ValueError(f"scaling kind must be one of {[k for k in takes if k]}")
        optional = ("fast", "slow", "attention_factor") if kind == "yarn" else ()
        missing = [k for k in takes[kind] if sc.get(k) is None]
        extra = [k for k in sc if k not in takes[kind] + optional]
        if missing or extra:
            raise ValueError(f"scaling {kind!r}: missing {missing}, not known {extra}")
        sc = {k: float(v) for k, v in sc.items() if v is not None}
        for k, v in sc.items():
            if not (v > 0.0 and math.isfinite(v)):
                raise ValueError(f"scaling {kind!r}: {k} must be positive and finite")
        i = np.arange(0, r, 2, dtype=np.float64)
        f = sc.get("factor", 1.0)
        if kind == "ntk":
            if r <= 2:
                raise ValueError("scaling 'ntk' needs rotary_dim > 2")
            theta = theta * f ** (r / (r - 2))
        inv = theta ** (-i / r) if r else i
        if kind == "linear":
            inv = inv / f
        elif kind == "bands":
            if not sc["high"] > sc["low"]:
                raise ValueError("scaling 'bands' needs high > low")
            turns = sc["original"] * inv / (2.0 * math.pi)
            keep = np.clip((turns - sc["low"]) / (sc["high"] - sc["low"]), 0.0, 1.0)
            inv = inv * (keep + (1.0 - keep) / f)
        elif kind == "yarn":
            if not theta > 1.0:
                raise ValueError("scaling 'yarn' needs theta > 1")

            def pair(turns):  # the (fractional) pair that makes so many turns
                return (r * math.log(sc["original"] / (turns * 2.0 * math.pi))
                        / (2.0 * math.log(theta)))

            lo = max(math.floor(pair(sc.get("fast", 32.0))), 0)
            hi = min(math.ceil(pair(sc.get("slow", 1.0))), r - 1)
            ramp = np.clip((i / 2 - lo) / max(hi - lo, 0.001), 0.0, 1.0)
            inv = inv * (1.0 - ramp) + inv / f * ramp
            return inv, sc.get("attention_factor", 0.1 * math.log(f) + 1.0)
        return inv, 1.0

    def to(self, device) -> "Rotary":
        """The same frequencies on `device` (itself if they are there)."""
        if self.turns.device == torch.device(device):
            return self
        r = Rotary.__new__(Rotary)
        r.__dict__.update(self.__dict__)
        r.turns = self.turns.to(device)
        return r


def _heads3(name: str, x: torch.Tensor, T: int, D: int):
    """(heads, stride of tokens, stride of heads) of x [T, heads, D]."""
    shape = x.shape
    if len(shape) != 3 or shape[0] != T or shape[2] != D:
        raise ValueError(f"{name} must be [T, heads, D] with T = {T}, D = {D}")
    st, sh, se = x.stride()
    if se != 1 and x.numel():
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return shape[1], st, sh


def qk_norm_rope_kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                    rotary: Optional[Rotary], k_pool: torch.Tensor, v_pool: torch.Tensor,
                    block_tables: torch.Tensor, base_lens: torch.Tensor, *, layer: int = 0,
                    cu_seqlens: Optional[torch.Tensor] = None,
                    q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                    eps: float = 1e-6, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Norm the q and k heads, turn them by their positions, and write k and v
    into the pages (``cfa_qk_norm_rope_kv``).  Returns q_out [T, Hq, D].

    q [T, Hq, D], k and v [T, Hkv, D], bf16 or fp16, may be views of one
    projection (any strides of tokens and heads; elements contiguous; D a
    multiple of 8, at most 256); positions [T] int32; `rotary` None: no
    rotation.  q_norm / k_norm [D]: RMSNorm weights of each head, of q's dtype
    or fp32 (None: no norm).  All in fp32, rounded once.

    Token t of sequence b goes to slot base_lens[b] + j of `layer` in k_pool /
    v_pool [num_blocks, num_layers, Hkv, block_size, D] by block_tables [B,
    max_blocks] int32: without cu_seqlens the T tokens are T / B per sequence,
    with it (int32 [B + 1], rising) token t is number j = t - cu_seqlens[b].
    Tokens that belong to no sequence leave every output as it was, and so do
    k and v whose page is not mapped (-1, or behind the table).
    q_out must not overlap q, k or v.
    """
    if not isinstance(q, torch.Tensor) or q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("q must be a bfloat16 or float16 tensor")
    dt, dev, shape = q.dtype, q.device, q.shape
    if len(shape) != 3:
        raise ValueError("q must be [T, Hq, D]")
    T, Hq, D = shape
    _require_all(dev, (("q", q, dt), ("k", k, dt), ("v", v, dt),
                       ("positions", positions, torch.int32), ("k_pool", k_pool, dt),
                       ("v_pool", v_pool, dt), ("block_tables", block_tables, torch.int32),
                       ("base_lens", base_lens, torch.int32)))
    _, q_st, q_sh = _heads3("q", q, T, D)
    Hkv, k_st, k_sh = _heads3("k", k, T, D)
    v_heads, v_st, v_sh = _heads3("v", v, T, D)
    if v_heads != Hkv:
        raise ValueError("k and v must have the same number of heads")
    if positions.shape != (T,):
        raise ValueError(f"positions must be [T] = [{T}]")
    for name, pool in (("k_pool", k_pool), ("v_pool", v_pool)):
        pools = pool.shape
        if len(pools) != 5 or not pool.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [blocks, layers, Hkv, block_size, D] tensor")
    if k_pool.shape != pools:
        raise ValueError("k_pool and v_pool must have the same shape")
    nblk, nlayers, ph, bs, pd = pools
    if ph != Hkv or pd != D:
        raise ValueError("the pools' heads and head_dim must be k's")
    tables, lens = block_tables.shape, base_lens.shape
    if len(lens) != 1 or len(tables) != 2 or tables[0] != lens[0]:
        raise ValueError("base_lens must be [B] and block_tables [B, max_blocks]")
    B = lens[0]
    if cu_seqlens is not None:
        _require_cuda("cu_seqlens", cu_seqlens, torch.int32, dev)
        if cu_seqlens.shape != (B + 1,):
            raise ValueError("cu_seqlens must be [B + 1]")
        cu_seqlens = cu_seqlens.contiguous()
    elif T and (B == 0 or T % B):
        raise ValueError("without cu_seqlens the tokens must be a multiple of the sequences")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is None:
            continue
        if not isinstance(w, torch.Tensor) or w.dtype not in (dt, torch.float32):
            raise ValueError(f"{name} must be {dt} or float32")
        _require_cuda(name, w, w.dtype, dev)
        if w.shape != (D,) or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [D] = [{D}]")
    if q_norm is not None and k_norm is not None and q_norm.dtype != k_norm.dtype:
        raise ValueError("q_norm and k_norm must have the same dtype")
    norm = q_norm if q_norm is not None else k_norm
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    rot = 0 if rotary is None else rotary.rotary_dim
    if rot > D:
        raise ValueError("rotary_dim exceeds the head's size")
    turns = None
    if rot:
        turns = rotary.turns
        _require_cuda("rotary.turns", turns, torch.int64, dev)
    if q_out is None:
        q_out = torch.empty(T, Hq, D, dtype=dt, device=dev)
    else:
        _require_cuda("q_out", q_out, dt, dev)
        if q_out.shape != shape or not q_out.is_contiguous():
            raise ValueError("q_out must be a contiguous [T, Hq, D]")
        lo = q_out.data_ptr()
        hi = lo + 2 * T * Hq * D
        for name, x, h, st, sh in (("q", q, Hq, q_st, q_sh), ("k", k, Hkv, k_st, k_sh),
                                   ("v", v, Hkv, v_st, v_sh)):
            at = x.data_ptr()
            if hi > at and at + 2 * ((T - 1) * st + (h - 1) * sh + D) > lo and T:
                raise ValueError(f"q_out must not overlap {name}")
    positions = positions.contiguous()
    block_tables = block_tables.contiguous()
    base_lens = base_lens.contiguous()
    with _on(dev):
        rc = _lib.load().cfa_qk_norm_rope_kv(
            q.data_ptr(), q_st, q_sh, k.data_ptr(), k_st, k_sh, v.data_ptr(), v_st, v_sh,
            dt == torch.float16, positions.data_ptr(), T, B, _ptr(cu_seqlens), Hq, Hkv, D, rot,
            _ptr(turns), rotary.factor if rot else 1.0,
            rot > 0 and rotary.layout == "interleaved", _ptr(q_norm), _ptr(k_norm),
            norm is not None and norm.dtype == torch.float32, eps, q_out.data_ptr(),
            k_pool.data_ptr(), v_pool.data_ptr(), nblk, nlayers, int(layer), bs,
            block_tables.data_ptr(), tables[1], base_lens.data_ptr(), _stream_ptr(dev))
    _lib.check(rc, "cfa_qk_norm_rope_kv")
    return q_out

