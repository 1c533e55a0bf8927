"""Tensor-level entry points of the verification path (PyTorch-ROCm host side).

Each function validates shapes, dtypes, devices and strides on the host,
allocates outputs and workspace with torch's caching allocator, and calls one
C-ABI entry point of ``libcfa.so`` on torch's current HIP stream.  Nothing here
computes on the CPU: without the HIP library every call raises.

Reference semantics (paths inside Bahaa-Labs/CUDAForge):
  chain_verify, mode="cpp"     csrc/src/scheduler/speculative.cpp:50-103
  chain_verify, mode="greedy"  csrc/src/scheduler/speculative.cpp:105-150
  chain_verify, mode="python"  cudaforge/speculative.py:152-195
  tree_attention               paged layout of csrc/src/memory/paged_kv_cache.cpp:
                               13-21, 409-421; descriptor of paged_kv_cache.h:81-94
  prompt_attention             dense causal attention of csrc/kernels/cuda/
                               flash_attn_v2.cu:45-195, over the paged layout
  kv_commit                    device half of append_tokens, paged_kv_cache.cpp:255-286
  kv_gather                    rows of the paged layout, read back token by token
  tree_verify                  speculative.cpp:50-150 generalised to a draft tree
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib

_MODES = {"cpp": _lib.CFA_MODE_CPP, "python": _lib.CFA_MODE_PYTHON, "greedy": _lib.CFA_MODE_GREEDY}
_KINDS = {"probs": _lib.CFA_INPUT_PROBS, "logits": _lib.CFA_INPUT_LOGITS}


def _stream_ptr(device: torch.device) -> int:
    # the raw handle, without a torch.cuda.Stream object for every call
    index = torch.cuda.current_device() if device.index is None else device.index
    return torch._C._cuda_getCurrentRawStream(index)


class _Here:
    """A context that changes nothing."""

    def __enter__(self):
        return self

    def __exit__(self, *a):
        return False


_HERE = _Here()


def _on(device: torch.device):
    """torch.cuda.device(device), or nothing where it is the current one (the
    usual case: entering it costs about 2 us of a call's 15)."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _require_cuda(name: str, t: torch.Tensor, dtype: torch.dtype, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    # (the usual case, in a third of the time that the checks by name take)
    if t.is_cuda and t.dtype is dtype and (device is None or t.get_device() == device.index):
        return
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a HIP device tensor (got {t.device})")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} (got {t.dtype})")


def _require_all(device: torch.device, named) -> None:
    """_require_cuda of each (name, tensor, dtype) on `device`, in half its time
    where all is well."""
    index = device.index
    try:
        for _, t, dtype in named:
            if t.dtype is not dtype or t.get_device() != index:
                break
        else:
            if index is not None and device.type == "cuda":
                return
    except AttributeError:
        pass
    for name, t, dtype in named:
        _require_cuda(name, t, dtype, device)


def _workspace(workspace: Optional[torch.Tensor], need: int, device: torch.device) -> torch.Tensor:
    """The caller's workspace where it holds `need` bytes, else a new one; one that
    lies elsewhere is refused (its address would be written to as if on `device`)."""
    if workspace is not None:
        _require_cuda("workspace", workspace, getattr(workspace, "dtype", None), device)
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        if workspace.numel() >= need:
            return workspace
    return torch.empty(max(need, 1), dtype=torch.uint8, device=device)


@dataclass
class ChainVerifyOutput:
    """Per-sequence results of one chain verification (all int32 device tensors).

    accept_len   [B]      accepted draft tokens (python mode: the batch-wide n)
    tokens       [B, K+1] accepted drafts then the final token, -1 padded
    num_emitted  [B]      valid entries of ``tokens``
    final        [B]      the resampled or bonus token (final_token)
    eos          [B]      end_of_sequence flag (cpp / greedy modes)
    target_probs / draft_probs  the fp32 probabilities the decisions used, when
                          ``return_probs`` was set
    """

    accept_len: torch.Tensor
    tokens: torch.Tensor
    num_emitted: torch.Tensor
    final: torch.Tensor
    eos: torch.Tensor
    target_probs: Optional[torch.Tensor] = None
    draft_probs: Optional[torch.Tensor] = None


def chain_workspace_bytes(B: int, K: int, V: int, input_kind: str = "logits",
                          mode: str = "cpp") -> int:
    return int(_lib.load().cfa_chain_verify_workspace_size(B, K, V, _KINDS[input_kind],
                                                            _MODES[mode]))


def chain_verify(target: torch.Tensor, draft: Optional[torch.Tensor],
                 draft_tokens: torch.Tensor, uniforms: Optional[torch.Tensor], *,
                 input_kind: str = "logits", temperature: float = 1.0, top_p: float = 1.0,
                 mode: str = "cpp", eos_token_id: int = -1, return_probs: bool = False,
                 workspace: Optional[torch.Tensor] = None) -> ChainVerifyOutput:
    """Verify B chains of K draft tokens in one pass over the logits.

    target [B, K+1, V] fp32 and draft [B, K, V] fp32 (None in greedy mode) may be
    strided views (the last dimension must be contiguous); draft_tokens [B, K]
    int32; uniforms fp32 in [0, 1): [B, K+1] in cpp mode, [B, K+2] in python
    mode (column K+1 drives the bonus that follows a rejection at the last
    position, speculative.py:188), None in greedy mode.

    input_kind "logits": probabilities are softmax(row / temperature), fused
    into the kernel; "probs": rows are probabilities (temperature unused).
    """
    if mode not in _MODES:
        raise ValueError(f"mode must be one of {sorted(_MODES)}")
    if input_kind not in _KINDS:
        raise ValueError(f"input_kind must be one of {sorted(_KINDS)}")
    _require_cuda("target", target, torch.float32)
    dev = target.device
    if target.dim() != 3:
        raise ValueError("target must be [B, K+1, V]")
    B, K1, V = target.shape
    K = K1 - 1
    if B <= 0 or V <= 0 or K < 0:
        raise ValueError("target must be [B, K+1, V] with B, V > 0")
    if target.stride(2) != 1:
        raise ValueError("target's vocabulary dimension must be contiguous")
    _require_cuda("draft_tokens", draft_tokens, torch.int32, dev)
    if tuple(draft_tokens.shape) != (B, K):
        raise ValueError(f"draft_tokens must be [B, K] = [{B}, {K}]")
    draft_tokens = draft_tokens.contiguous()
    greedy = mode == "greedy"
    if not greedy:
        if draft is None or uniforms is None:
            raise ValueError("draft and uniforms are required outside greedy mode")
        _require_cuda("draft", draft, torch.float32, dev)
        if tuple(draft.shape) != (B, K, V):
            raise ValueError("Incompatible draft and target tensor dimensions in SpeculativeEngine.")
        if K > 0 and draft.stride(2) != 1:
            raise ValueError("draft's vocabulary dimension must be contiguous")
        _require_cuda("uniforms", uniforms, torch.float32, dev)
        nu = K + 2 if mode == "python" else K + 1
        if tuple(uniforms.shape) != (B, nu):
            cols = "K+2" if mode == "python" else "K+1"
            raise ValueError(f"uniforms must be [B, {cols}] = [{B}, {nu}] in {mode} mode")
        uniforms = uniforms.contiguous()
    if input_kind == "logits" and not temperature > 0.0:
        raise ValueError("temperature must be > 0")

    lib = _lib.load()
    ws_need = int(lib.cfa_chain_verify_workspace_size(B, K, V, _KINDS[input_kind], _MODES[mode]))
    if workspace is None or workspace.numel() < ws_need:
        workspace = torch.empty(max(ws_need, 1), dtype=torch.uint8, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    out = ChainVerifyOutput(
        accept_len=torch.empty(B, **i32), tokens=torch.empty(B, K + 1, **i32),
        num_emitted=torch.empty(B, **i32), final=torch.empty(B, **i32),
        eos=torch.empty(B, **i32))
    if return_probs:
        out.target_probs = torch.empty(B, K + 1, V, dtype=torch.float32, device=dev)
        if not greedy and K > 0:
            out.draft_probs = torch.empty(B, K, V, dtype=torch.float32, device=dev)
    d_sb = d_sk = 0
    if draft is not None and not greedy:
        d_sb, d_sk = draft.stride(0), draft.stride(1)
        if K == 0:
            d_sb = d_sk = V
    with torch.cuda.device(dev):
        rc = lib.cfa_chain_verify(
            target.data_ptr(), target.stride(0), target.stride(1),
            None if greedy or draft is None else draft.data_ptr(), d_sb, d_sk,
            _KINDS[input_kind], draft_tokens.data_ptr(),
            None if uniforms is None else uniforms.data_ptr(),
            B, K, V, ctypes.c_float(temperature), ctypes.c_float(top_p), _MODES[mode],
            int(eos_token_id), out.accept_len.data_ptr(), out.tokens.data_ptr(),
            out.num_emitted.data_ptr(), out.final.data_ptr(), out.eos.data_ptr(),
            _ptr(out.target_probs), _ptr(out.draft_probs), workspace.data_ptr(),
            workspace.numel(), _stream_ptr(dev))
    _lib.check(rc, "cfa_chain_verify")
    return out


def tree_attention_workspace_bytes(B: int, N: int, n_q_heads: int, n_kv_heads: int,
                                   head_dim: int, max_keys: int, num_splits: int = 0, *,
                                   scored: bool = False, window: int = 0, sinks: int = 0,
                                   e4m3: bool = False) -> int:
    """Workspace of ``tree_attention`` for N query nodes; `scored`: with a cap,
    a bias, a window or fp16 tensors; `e4m3`: over pools with scales."""
    if scored or window or e4m3:
        return int(_lib.load().cfa_tree_attention_cached_workspace_size(
            B, N, n_q_heads, n_kv_heads, head_dim, _int32(max_keys), _int32(window), _int32(sinks),
            int(e4m3), num_splits))
    return int(_lib.load().cfa_tree_attention_workspace_size(B, N, n_q_heads, n_kv_heads,
                                                              head_dim, max_keys, num_splits))


def _half_dtype(q) -> torch.dtype:
    """bfloat16, or float16 where q is."""
    is_half = isinstance(q, torch.Tensor) and q.dtype == torch.float16
    return torch.float16 if is_half else torch.bfloat16


def _check_pools(k_pool: torch.Tensor, v_pool: torch.Tensor, D: int):
    for name, pool in (("k_pool", k_pool), ("v_pool", v_pool)):
        if pool.dim() != 5 or not pool.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [blocks, layers, Hkv, block_size, D] tensor")
    if k_pool.shape != v_pool.shape:
        raise ValueError("k_pool and v_pool must have the same shape")
    if k_pool.shape[4] != D:
        raise ValueError("head_dim of q and of the pools differ")


def _cache_dtype(k_scales, v_scales, dtype: torch.dtype) -> torch.dtype:
    """The pools' type: e4m3 where there are scales, else `dtype`."""
    if (k_scales is None) != (v_scales is None):
        raise ValueError("k_scales and v_scales go together")
    return dtype if k_scales is None else torch.float8_e4m3fn


def _check_scales(k_scales, v_scales, pools, dev) -> None:
    """The scales of e4m3 pools of that shape (None: 16-bit pools)."""
    for name, s in (("k_scales", k_scales), ("v_scales", v_scales)):
        if s is None:
            continue
        _require_cuda(name, s, torch.uint8, dev)
        if s.shape != pools[:4] or not s.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [blocks, layers, Hkv, block_size]")


def _check_slopes(alibi_slopes: Optional[torch.Tensor], Hq: int, dev) -> Optional[torch.Tensor]:
    if alibi_slopes is None:
        return None
    _require_cuda("alibi_slopes", alibi_slopes, torch.float32, dev)
    if tuple(alibi_slopes.shape) != (Hq,):
        raise ValueError(f"alibi_slopes must be [Hq] = [{Hq}]")
    return alibi_slopes.contiguous()


def _int32(n: int) -> int:
    """A bound as the entry points take it: past every position, the largest is the
    same (a wider one would lose its upper bits on the way)."""
    return min(int(n), 2 ** 31 - 1)


def _aligned(q: torch.Tensor) -> torch.Tensor:
    """q, or a copy of it where it does not begin on 16 bytes."""
    return q if q.data_ptr() % 16 == 0 else q.clone()


def _check_out(out: Optional[torch.Tensor], q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q)
    _require_cuda("out", out, q.dtype, q.device)
    if out.shape != q.shape or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape")
    if out.data_ptr() % 16:
        raise ValueError("out must be 16-byte aligned")
    return out


def tree_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                   block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                   tree_mask: torch.Tensor, *, layer: int = 0,
                   sm_scale: Optional[float] = None, max_keys: Optional[int] = None,
                   num_splits: int = 0, out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None, first_node: int = 0,
                   soft_cap: float = 0.0, alibi_slopes: Optional[torch.Tensor] = None,
                   window: int = 0, sinks: int = 0, k_scales: Optional[torch.Tensor] = None,
                   v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Tree-masked attention of draft-tree nodes over a paged KV cache.

    q [B, Nq, Hq, D] bf16 (D = 128 or 64): the queries of tree nodes
    first_node .. first_node + Nq - 1 of an N = first_node + Nq node tree;
    k_pool / v_pool [num_blocks, num_layers, Hkv, block_size, D] bf16 (the
    reference's per-block layout); block_tables [B, max_blocks] int32;
    ctx_lens [B] int32 (tokens before the tree; the tree's K/V sit at
    ctx_len + i, i < N); tree_mask int64 [N] or [B, N] holding each node's
    64-bit ancestor-or-self mask.  max_keys bounds ctx_len + N on the host
    (computed with one sync when omitted).  Returns [B, Nq, Hq, D] bf16.

    A tree of one node (tree_mask [1] holding 1) is plain decode.

    Scores of other decoders (``cfa_tree_attention_cached``): soft_cap > 0
    takes cap * tanh(s / cap) of each scaled score; alibi_slopes [Hq] fp32
    subtracts slope * distance, where a node stands at ctx_len + its depth (the
    bits of its mask less one); window > 0 hides keys at a distance of window
    and more, but those in a sequence's first `sinks` slots.  q and the pools may
    then be fp16, and Hq / Hkv * Nq may exceed 256; fp16 tensors take this path by
    themselves.  A query that sees no key gets zeros.

    With k_scales and v_scales (uint8 [num_blocks, num_layers, Hkv, block_size])
    the pools are float8_e4m3fn, as ``rotary.qk_norm_rope_kv`` writes them; q is
    bf16 or fp16, and keys and values are taken in its type.
    """
    dtype = _half_dtype(q)
    _require_cuda("q", q, dtype)
    dev = q.device
    if q.dim() != 4:
        raise ValueError("q must be [B, Nq, Hq, D]")
    B, Nq, Hq, D = q.shape
    if first_node < 0:
        raise ValueError("first_node must be >= 0")
    N = first_node + Nq
    q = q.contiguous()
    cache = _cache_dtype(k_scales, v_scales, dtype)
    _require_all(dev, (("k_pool", k_pool, cache), ("v_pool", v_pool, cache),
                       ("block_tables", block_tables, torch.int32),
                       ("ctx_lens", ctx_lens, torch.int32), ("tree_mask", tree_mask, torch.int64)))
    _check_pools(k_pool, v_pool, D)
    nblk, nlayers, Hkv, bs, _ = k_pool.shape
    _check_scales(k_scales, v_scales, k_pool.shape, dev)
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    if block_tables.dim() != 2 or block_tables.shape[0] != B:
        raise ValueError("block_tables must be [B, max_blocks]")
    block_tables = block_tables.contiguous()
    if tuple(ctx_lens.shape) != (B,):
        raise ValueError("ctx_lens must be [B]")
    ctx_lens = ctx_lens.contiguous()
    if tree_mask.dim() == 1 and tree_mask.shape[0] == N:
        mstride = 0
    elif tree_mask.dim() == 2 and tuple(tree_mask.shape) == (B, N):
        mstride = N
    else:
        raise ValueError("tree_mask must be [N] or [B, N]")
    tree_mask = tree_mask.contiguous()
    if sm_scale is None:
        sm_scale = D ** -0.5
    if max_keys is None:
        max_keys = int(ctx_lens.max().item()) + N
    e4m3 = k_scales is not None
    scored = (soft_cap != 0.0 or alibi_slopes is not None or window != 0
              or dtype == torch.float16 or e4m3)
    if scored:
        window, sinks, max_keys = _int32(window), _int32(sinks), _int32(max_keys)
        alibi_slopes = _check_slopes(alibi_slopes, Hq, dev)
        q = _aligned(q)
        out = _check_out(out, q)
    elif out is None:
        out = torch.empty_like(q)
    lib = _lib.load()
    with _on(dev):
        if scored:
            need = int(lib.cfa_tree_attention_cached_workspace_size(
                B, Nq, Hq, Hkv, D, max_keys, window, sinks, e4m3, num_splits))
        else:
            need = int(lib.cfa_tree_attention_workspace_size(B, Nq, Hq, Hkv, D, max_keys,
                                                             num_splits))
        workspace = _workspace(workspace, need, dev)
        if scored:
            rc = lib.cfa_tree_attention_cached(
                q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), _ptr(k_scales),
                _ptr(v_scales), int(dtype == torch.float16), block_tables.data_ptr(),
                block_tables.shape[1], ctx_lens.data_ptr(), nblk, nlayers, int(layer), bs,
                tree_mask.data_ptr(), mstride, B, N, int(first_node), Hq, Hkv, D, sm_scale,
                soft_cap, _ptr(alibi_slopes), window, sinks, max_keys, int(num_splits),
                out.data_ptr(), workspace.data_ptr(), workspace.numel(), _stream_ptr(dev))
        else:
            rc = lib.cfa_tree_attention(
                q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), block_tables.data_ptr(),
                block_tables.shape[1], ctx_lens.data_ptr(), nblk, nlayers, int(layer), bs,
                tree_mask.data_ptr(), mstride, B, N, int(first_node), Hq, Hkv, D,
                sm_scale, int(max_keys), int(num_splits), out.data_ptr(),
                workspace.data_ptr(), workspace.numel(), _stream_ptr(dev))
    _lib.check(rc, "cfa_tree_attention_cached" if scored else "cfa_tree_attention")
    return out


def prompt_attention_workspace_bytes(T: int, B: int, n_q_heads: int, n_kv_heads: int,
                                     head_dim: int, max_query: int, max_keys: int,
                                     window: int = 0, num_splits: int = 0, *, sinks: int = 0,
                                     e4m3: bool = False) -> int:
    return int(_lib.load().cfa_prompt_attention_cached_workspace_size(
        T, B, n_q_heads, n_kv_heads, head_dim, _int32(max_query), _int32(max_keys), _int32(window),
        _int32(sinks), int(e4m3), num_splits))


def prompt_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                     block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                     cu_seqlens: torch.Tensor, *, layer: int = 0,
                     sm_scale: Optional[float] = None, max_query: Optional[int] = None,
                     max_keys: Optional[int] = None, soft_cap: float = 0.0,
                     alibi_slopes: Optional[torch.Tensor] = None, window: int = 0,
                     num_splits: int = 0, out: Optional[torch.Tensor] = None,
                     workspace: Optional[torch.Tensor] = None, sinks: int = 0,
                     k_scales: Optional[torch.Tensor] = None,
                     v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of prompt chunks over a paged KV cache
    (``cfa_prompt_attention_cached``).

    q [T, Hq, D] (bf16 or fp16, D = 128 or 64) holds B sequences' new tokens one
    after another: cu_seqlens int32 [B + 1] says where each begins.  ctx_lens
    [B] int32 are the tokens in front of each chunk (0 for a first one); the
    chunk's own K and V are in the pages already (``rotary.qk_norm_rope_kv``),
    and token i of it sees the slots up to ctx_len + i.  Pools, block_tables,
    soft_cap, alibi_slopes, window, sinks, k_scales and v_scales are those of
    ``tree_attention``.
    max_query and max_keys are guesses of the longest chunk and of the largest
    ctx_len + chunk (default T and the tables' capacity): they plan the call,
    and any positive values are right.  Rows of q behind the last sequence get
    no output: `out` keeps what it had there.  Tokens behind a table's last page
    see what the table covers.  Returns out [T, Hq, D].
    """
    dtype = _half_dtype(q)
    _require_cuda("q", q, dtype)
    dev = q.device
    if q.dim() != 3:
        raise ValueError("q must be [T, Hq, D]")
    T, Hq, D = q.shape
    q = q.contiguous()
    cache = _cache_dtype(k_scales, v_scales, dtype)
    _require_all(dev, (("k_pool", k_pool, cache), ("v_pool", v_pool, cache),
                       ("ctx_lens", ctx_lens, torch.int32),
                       ("block_tables", block_tables, torch.int32),
                       ("cu_seqlens", cu_seqlens, torch.int32)))
    _check_pools(k_pool, v_pool, D)
    nblk, nlayers, Hkv, bs, _ = k_pool.shape
    _check_scales(k_scales, v_scales, k_pool.shape, dev)
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    if ctx_lens.dim() != 1:
        raise ValueError("ctx_lens must be [B]")
    B = ctx_lens.shape[0]
    if block_tables.dim() != 2 or block_tables.shape[0] != B:
        raise ValueError("block_tables must be [B, max_blocks]")
    if tuple(cu_seqlens.shape) != (B + 1,):
        raise ValueError("cu_seqlens must be [B + 1]")
    block_tables, ctx_lens, cu_seqlens = (t.contiguous() for t in
                                          (block_tables, ctx_lens, cu_seqlens))
    alibi_slopes = _check_slopes(alibi_slopes, Hq, dev)
    q = _aligned(q)
    out = _check_out(out, q)
    if sm_scale is None:
        sm_scale = D ** -0.5
    window, sinks = _int32(window), _int32(sinks)
    max_query = _int32(max(T, 1) if max_query is None else max_query)
    max_keys = _int32(max(block_tables.shape[1] * bs, 1) if max_keys is None else max_keys)
    lib = _lib.load()
    with _on(dev):
        need = int(lib.cfa_prompt_attention_cached_workspace_size(
            T, B, Hq, Hkv, D, max_query, max_keys, window, sinks, k_scales is not None,
            num_splits))
        workspace = _workspace(workspace, need, dev)
        rc = lib.cfa_prompt_attention_cached(
            q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), _ptr(k_scales), _ptr(v_scales),
            int(dtype == torch.float16),
            block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(), nblk, nlayers,
            int(layer), bs, cu_seqlens.data_ptr(), T, B, Hq, Hkv, D, sm_scale, soft_cap,
            _ptr(alibi_slopes), window, sinks, max_query, max_keys, int(num_splits),
            out.data_ptr(), workspace.data_ptr(), workspace.numel(), _stream_ptr(dev))
    _lib.check(rc, "cfa_prompt_attention_cached")
    return out


@dataclass
class KVCommitOutput:
    new_ctx_lens: torch.Tensor  # [B] int32: ctx_lens + path_len (unchanged when rejected)
    status: torch.Tensor        # [B] int32: 0 committed, 1 rejected (bad path or page)


def kv_commit(k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
              ctx_lens: torch.Tensor, paths: torch.Tensor, path_lens: torch.Tensor, *,
              k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None
              ) -> KVCommitOutput:
    """Move each sequence's accepted tree nodes (paths [B, P] int32, node ids
    with the root 0 first, path_lens [B]) from slots ctx + node to ctx + j in
    every layer and KV head of both pools (in place).  Of e4m3 pools the rows'
    scales (uint8 [num_blocks, num_layers, Hkv, block_size]) move with them."""
    for name, pool in (("k_pool", k_pool), ("v_pool", v_pool)):
        if not isinstance(pool, torch.Tensor) or pool.device.type != "cuda":
            raise ValueError(f"{name} must be a HIP device tensor")
        if pool.dim() != 5 or not pool.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [blocks, layers, Hkv, block_size, D] tensor")
    if k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype:
        raise ValueError("k_pool and v_pool must match in shape and dtype")
    dev = k_pool.device
    if v_pool.device != dev:
        raise ValueError("k_pool and v_pool must be on the same device")
    if _cache_dtype(k_scales, v_scales, k_pool.dtype) != k_pool.dtype:
        raise ValueError("k_scales and v_scales go with float8_e4m3fn pools")
    _check_scales(k_scales, v_scales, k_pool.shape, dev)
    nblk, nlayers, Hkv, bs, D = k_pool.shape
    _require_cuda("block_tables", block_tables, torch.int32, dev)
    B = block_tables.shape[0]
    for name, t, shape in (("ctx_lens", ctx_lens, (B,)), ("path_lens", path_lens, (B,))):
        _require_cuda(name, t, torch.int32, dev)
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must be [B]")
    _require_cuda("paths", paths, torch.int32, dev)
    if paths.dim() != 2 or paths.shape[0] != B:
        raise ValueError("paths must be [B, max_path]")
    block_tables, ctx_lens, paths, path_lens = (t.contiguous() for t in
                                                (block_tables, ctx_lens, paths, path_lens))
    out = KVCommitOutput(new_ctx_lens=torch.empty(B, dtype=torch.int32, device=dev),
                         status=torch.empty(B, dtype=torch.int32, device=dev))
    with torch.cuda.device(dev):
        rc = _lib.load().cfa_kv_commit_scaled(
            k_pool.data_ptr(), v_pool.data_ptr(), _ptr(k_scales), _ptr(v_scales),
            block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(), paths.data_ptr(),
            paths.shape[1], path_lens.data_ptr(), B, nblk, nlayers, Hkv, bs, D,
            k_pool.element_size(), out.new_ctx_lens.data_ptr(), out.status.data_ptr(),
            _stream_ptr(dev))
    _lib.check(rc, "cfa_kv_commit")
    return out


def kv_gather(k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
              starts: torch.Tensor, *, tokens: Optional[int] = None, layer: int = 0,
              cu_seqlens: Optional[torch.Tensor] = None,
              k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
              dtype: Optional[torch.dtype] = None, k_out: Optional[torch.Tensor] = None,
              v_out: Optional[torch.Tensor] = None):
    """Read sequences' keys and values back out of their pages
    (``cfa_kv_gather``).  Returns (k, v), each [T, Hkv, D].

    Token j of sequence b is the row at slot starts[b] + j (starts [B] int32)
    of `layer`, by block_tables [B, max_blocks] int32: without cu_seqlens the T
    tokens are T / B per sequence, with it (int32 [B + 1], rising) token t is
    number j = t - cu_seqlens[b].  T is k_out's, or `tokens`.  e4m3 pools
    [num_blocks, num_layers, Hkv, block_size, D] with k_scales and v_scales
    (uint8, their first four dimensions; ``rotary.qk_norm_rope_kv`` fills both)
    give the values that the codes stand for, in `dtype` or the outputs' (bf16,
    exact, or fp16, rounded once); bf16 and fp16 pools are copied.  D is a
    multiple of 16, at most 256.

    Tokens whose page is not mapped (-1, or behind the table) are zeros.  Rows
    of no sequence keep what k_out and v_out had there (zeros without those).
    """
    if not isinstance(k_pool, torch.Tensor) or k_pool.device.type != "cuda":
        raise ValueError("k_pool must be a HIP device tensor")
    dev = k_pool.device
    if (k_out is None) != (v_out is None):
        raise ValueError("k_out and v_out go together")
    if dtype is None:
        if isinstance(k_out, torch.Tensor):
            dtype = k_out.dtype
        else:
            dtype = torch.bfloat16 if k_scales is not None else k_pool.dtype
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("the outputs must be bfloat16 or float16")
    cache = _cache_dtype(k_scales, v_scales, dtype)
    _require_all(dev, (("k_pool", k_pool, cache), ("v_pool", v_pool, cache),
                       ("block_tables", block_tables, torch.int32),
                       ("starts", starts, torch.int32)))
    if k_pool.dim() != 5:
        raise ValueError("k_pool must be [blocks, layers, Hkv, block_size, D]")
    nblk, nlayers, Hkv, bs, D = k_pool.shape
    _check_pools(k_pool, v_pool, D)
    _check_scales(k_scales, v_scales, k_pool.shape, dev)
    if starts.dim() != 1 or block_tables.dim() != 2 or block_tables.shape[0] != starts.shape[0]:
        raise ValueError("starts must be [B] and block_tables [B, max_blocks]")
    B = starts.shape[0]
    if k_out is not None:
        T = k_out.shape[0] if isinstance(k_out, torch.Tensor) and k_out.dim() else -1
        if tokens not in (None, T):
            raise ValueError("tokens differs from k_out's")
        for name, t in (("k_out", k_out), ("v_out", v_out)):
            _require_cuda(name, t, dtype, dev)
            if tuple(t.shape) != (T, Hkv, D) or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be a contiguous, 16-byte aligned [T, Hkv, D]")
        if abs(k_out.data_ptr() - v_out.data_ptr()) < 2 * T * Hkv * D:
            raise ValueError("k_out and v_out must not overlap")
    else:
        if tokens is None:
            raise ValueError("give tokens, or k_out and v_out")
        T = int(tokens)
        if T < 0:
            raise ValueError("tokens must not be negative")
    if cu_seqlens is not None:
        _require_cuda("cu_seqlens", cu_seqlens, torch.int32, dev)
        if tuple(cu_seqlens.shape) != (B + 1,):
            raise ValueError("cu_seqlens must be [B + 1]")
        cu_seqlens = cu_seqlens.contiguous()
    elif T and (B == 0 or T % B):
        raise ValueError("without cu_seqlens the tokens must be a multiple of the sequences")
    if k_out is None:
        new = torch.empty if cu_seqlens is None else torch.zeros
        k_out, v_out = (new(T, Hkv, D, dtype=dtype, device=dev) for _ in range(2))
    block_tables, starts = block_tables.contiguous(), starts.contiguous()
    with _on(dev):
        rc = _lib.load().cfa_kv_gather(
            k_pool.data_ptr(), v_pool.data_ptr(), _ptr(k_scales), _ptr(v_scales),
            dtype == torch.float16, nblk, nlayers, int(layer), Hkv, bs, D,
            block_tables.data_ptr(), block_tables.shape[1], starts.data_ptr(), _ptr(cu_seqlens),
            T, B, k_out.data_ptr(), v_out.data_ptr(), _stream_ptr(dev))
    _lib.check(rc, "cfa_kv_gather")
    return k_out, v_out


@dataclass
class TreeVerifyOutput:
    """Per-sequence results of tree verification (int32 device tensors)."""

    path: torch.Tensor         # [B, N] accepted node ids from the root, -1 padded
    path_len: torch.Tensor     # [B] 1 + accepted drafts
    tokens: torch.Tensor       # [B, N+1] accepted draft tokens then the final token
    num_emitted: torch.Tensor  # [B]
    final: torch.Tensor        # [B]
    eos: torch.Tensor          # [B]
    status: torch.Tensor       # [B] 0 ok, 1 uniforms ran out, 2 a team wait timed out
    target_probs: Optional[torch.Tensor] = None
    draft_probs: Optional[torch.Tensor] = None

    def check_status(self) -> None:
        """Raise RuntimeError unless every sequence's status is 0 (one host sync)."""
        check_status(self.status)


TREE_STATUS = {1: "the uniform stream ran out",
               2: "a wait between the work-groups of its team timed out (kernels of other "
                  "streams held a member back); run the call again"}


def check_status(status: torch.Tensor) -> None:
    """Raise RuntimeError when a tree verification reported a failure.

    status [B] int32 (``TreeVerifyOutput.status``): 0 ok, 1 the uniform
    stream ran out, 2 a team wait timed out.  The paths and tokens of a
    failed call are not valid and must not be committed; the reference raises
    rather than return unusable results (speculative.cpp:58-62).  Reads the
    status to the host: one synchronisation with its stream."""
    st = status.detach().to("cpu", torch.int32).reshape(-1)
    bad = torch.nonzero(st).reshape(-1).tolist()
    if not bad:
        return
    codes = sorted({int(st[b]) for b in bad})
    what = "; ".join(f"{TREE_STATUS.get(c, f'status {c}')} (sequences "
                     f"{[b for b in bad if int(st[b]) == c][:8]})" for c in codes)
    raise RuntimeError(f"cfa_tree_verify failed: {what}")


def tree_verify(target: torch.Tensor, draft: Optional[torch.Tensor], parents: torch.Tensor,
                node_tokens: torch.Tensor, uniforms: Optional[torch.Tensor], *,
                input_kind: str = "logits", temperature: float = 1.0, mode: str = "cpp",
                eos_token_id: int = -1, return_probs: bool = False,
                workspace: Optional[torch.Tensor] = None) -> TreeVerifyOutput:
    """Accept the longest root-to-leaf path of a draft tree.

    target / draft [B, N, V] fp32 (rows may be strided; the vocabulary
    dimension contiguous); parents [N] or [B, N] int32 with parents[c] < c and
    parents[0] = -1; node_tokens [B, N] int32; uniforms [B, n_u] fp32 (cpp mode).
    workspace: optional uint8 device tensor of tree_verify_workspace_bytes(B).
    status: 0 ok, 1 the uniform stream ran out, 2 a wait between the
    work-groups of a sequence timed out -- kernels of other streams held one
    of them back; run the call again.  ``check_status`` (or the output's
    ``check_status()``) raises RuntimeError on either; the call itself does
    not synchronise.
    """
    if mode not in ("cpp", "greedy"):
        raise ValueError("mode must be 'cpp' or 'greedy'")
    if input_kind not in _KINDS:
        raise ValueError(f"input_kind must be one of {sorted(_KINDS)}")
    _require_cuda("target", target, torch.float32)
    dev = target.device
    if target.dim() != 3 or target.stride(2) != 1:
        raise ValueError("target must be [B, N, V] with a contiguous last dimension")
    B, N, V = target.shape
    greedy = mode == "greedy"
    if not greedy:
        if draft is None or uniforms is None:
            raise ValueError("draft and uniforms are required in cpp mode")
        _require_cuda("draft", draft, torch.float32, dev)
        if tuple(draft.shape) != (B, N, V) or draft.stride(2) != 1:
            raise ValueError("draft must be [B, N, V] with a contiguous last dimension")
        _require_cuda("uniforms", uniforms, torch.float32, dev)
        if uniforms.dim() != 2 or uniforms.shape[0] != B:
            raise ValueError("uniforms must be [B, n_uniforms]")
        uniforms = uniforms.contiguous()
    _require_cuda("parents", parents, torch.int32, dev)
    if parents.dim() == 1 and parents.shape[0] == N:
        pstride = 0
    elif parents.dim() == 2 and tuple(parents.shape) == (B, N):
        pstride = N
    else:
        raise ValueError("parents must be [N] or [B, N]")
    parents = parents.contiguous()
    _require_cuda("node_tokens", node_tokens, torch.int32, dev)
    if tuple(node_tokens.shape) != (B, N):
        raise ValueError("node_tokens must be [B, N]")
    node_tokens = node_tokens.contiguous()
    if input_kind == "logits" and not temperature > 0.0:
        raise ValueError("temperature must be > 0")
    i32 = dict(dtype=torch.int32, device=dev)
    out = TreeVerifyOutput(path=torch.empty(B, N, **i32), path_len=torch.empty(B, **i32),
                           tokens=torch.empty(B, N + 1, **i32), num_emitted=torch.empty(B, **i32),
                           final=torch.empty(B, **i32), eos=torch.empty(B, **i32),
                           status=torch.empty(B, **i32))
    if return_probs:
        out.target_probs = torch.zeros(B, N, V, dtype=torch.float32, device=dev)
        if not greedy:
            out.draft_probs = torch.zeros(B, N, V, dtype=torch.float32, device=dev)
    lib = _lib.load()
    need = int(lib.cfa_tree_verify_workspace_size(B))
    if workspace is None or workspace.numel() < need or workspace.data_ptr() % 256:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        rc = lib.cfa_tree_verify(
            target.data_ptr(), target.stride(0), target.stride(1),
            None if greedy else draft.data_ptr(), 0 if greedy else draft.stride(0),
            0 if greedy else draft.stride(1), _KINDS[input_kind], parents.data_ptr(), pstride,
            node_tokens.data_ptr(), None if greedy else uniforms.data_ptr(),
            0 if greedy else uniforms.shape[1], B, N, V, ctypes.c_float(temperature),
            _MODES[mode], int(eos_token_id), out.path.data_ptr(), out.path_len.data_ptr(),
            out.tokens.data_ptr(), out.num_emitted.data_ptr(), out.final.data_ptr(),
            out.eos.data_ptr(), out.status.data_ptr(), _ptr(out.target_probs),
            _ptr(out.draft_probs), workspace.data_ptr(), workspace.numel(), _stream_ptr(dev))
    _lib.check(rc, "cfa_tree_verify")
    return out


def tree_verify_workspace_bytes(B: int) -> int:
    return int(_lib.load().cfa_tree_verify_workspace_size(B))
