"""Token sampling on the GPU: plain decode and draft-tree expansion.

Mirrors the reference's two samplers:

* ``fused_sampling_triton(logits, temperature)``
  (``csrc/kernels/triton/sampling_triton.py:40-66``): the argmax of
  ``softmax(logits / T)``, i.e. of the logits, first index on ties;
* ``launch_fused_sampling`` / ``fused_sampling_kernel``
  (``csrc/include/cudaforge/engine/sampling.h:18-28, 61-216``): temperature
  <= 1e-5 is greedy (first argmax of the raw logits), otherwise one
  multinomial draw per row from ``softmax(logits / T)`` by the sequential fp32
  inverse CDF ``cdf += p_i; if (u <= cdf)``, V - 1 if none.  The reference
  kernel takes ``top_k`` / ``top_p`` but never applies them; so does this
  mirror.  Its uniforms come from cuRAND Philox seeded with ``rng_seed``; here
  they come from torch's generator seeded with ``rng_seed`` (another stream)
  or from the caller.

``sample`` is the general entry point (``cfa_sample``): multinomial,
filtered (top-p keep rule of ``cudaforge/speculative.py:67-81`` plus top-k,
renormalised), or greedy top-k; several independent draws per row.
``expand_tree_level`` uses it to draw the children of draft-tree nodes.

``sample_rows`` (``cfa_sample_rows``) serves batches whose requests have their
own temperature, top-k, top-p and min-p; ``filtered_probs`` gives the same
rows' probabilities alone, for verification (``input_kind="probs"``).

``adjust_logits`` (``cfa_adjust_logits``) goes in front of any of them, and of
``verify.chain_verify`` and ``verify.tree_verify``: penalties of repeated tokens,
biases and grammar masks, of single rows and of a draft tree's nodes.

Every call runs on the HIP library; there is no CPU fallback.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .verify import _KINDS, _on, _ptr, _require_cuda, _stream_ptr, _workspace

__all__ = [
    "SamplingParams",
    "sample",
    "sample_workspace_bytes",
    "fused_sampling_triton",
    "launch_fused_sampling",
    "expand_tree_level",
    "sample_rows",
    "sample_rows_workspace_bytes",
    "filtered_probs",
    "adjust_logits",
]

_SMODES = {"multinomial": _lib.CFA_SAMPLE_MULTINOMIAL, "filtered": _lib.CFA_SAMPLE_FILTERED,
           "greedy": _lib.CFA_SAMPLE_GREEDY}


@dataclass
class SamplingParams:
    """sampling.h:18-28 (device pointers become tensors)."""

    logits: Optional[torch.Tensor] = None         # [batch_size, vocab_size]
    output_tokens: Optional[torch.Tensor] = None  # [batch_size] int32
    batch_size: int = 0
    vocab_size: int = 0
    temperature: float = 1.0
    top_k: int = 50
    top_p: float = 0.9
    rng_seed: int = 1337


def sample_workspace_bytes(R: int, V: int, draws: int = 1, mode: str = "multinomial") -> int:
    return int(_lib.load().cfa_sample_workspace_size(R, V, draws, _SMODES[mode]))


def _rows_f32(x: torch.Tensor) -> torch.Tensor:
    if x.dtype in (torch.float16, torch.bfloat16):
        x = x.float()
    if x.dim() != 2:
        raise ValueError("rows must be [R, V]")
    if x.stride(1) != 1:
        x = x.contiguous()
    return x


def sample(rows: torch.Tensor, *, mode: str = "multinomial", temperature: float = 1.0,
           top_k: int = -1, top_p: float = 1.0, draws: int = 1,
           uniforms: Optional[torch.Tensor] = None, generator: Optional[torch.Generator] = None,
           input_kind: str = "logits", return_probs: bool = False,
           workspace: Optional[torch.Tensor] = None):
    """Draw `draws` tokens from each of R rows ([R, V] logits or
    probabilities; fp32, or fp16/bf16 converted to fp32 first).

    mode "multinomial": softmax(row / T), sequential fp32 inverse CDF;
    "filtered": the top-p keep rule and top-k (<= 0: off), renormalised;
    "greedy": the `draws` largest values, largest first.  uniforms [R, draws]
    fp32 (drawn from `generator` when omitted: in (0, 1] for multinomial, in
    [0, 1) for filtered).  Returns int32
    [R, draws] (and the probabilities used, [R, V], with return_probs).
    """
    if mode not in _SMODES:
        raise ValueError(f"mode must be one of {sorted(_SMODES)}")
    if input_kind not in _KINDS:
        raise ValueError("input_kind must be 'logits' or 'probs'")
    if not isinstance(rows, torch.Tensor) or rows.device.type != "cuda":
        raise ValueError("rows must be a HIP device tensor")
    x = _rows_f32(rows)
    dev = x.device
    R, V = x.shape
    if draws < 1:
        raise ValueError("draws must be >= 1")
    out = torch.empty(R, draws, dtype=torch.int32, device=dev)
    probs = None
    u = None
    if mode != "greedy":
        if uniforms is None:
            u = torch.rand(R, draws, device=dev, generator=generator, dtype=torch.float32)
            if mode == "multinomial":
                # (0, 1], the range of curand_uniform: u = 0 would meet
                # `u <= cumulative` at index 0 whatever its probability
                # (the filtered draw takes the first prefix sum exceeding u
                # instead, so [0, 1) is right there)
                u = 1.0 - u
        else:
            _require_cuda("uniforms", uniforms, torch.float32, dev)
            if tuple(uniforms.shape) != (R, draws):
                raise ValueError("uniforms must be [R, draws]")
            u = uniforms.contiguous()
        if return_probs:
            probs = torch.empty(R, V, dtype=torch.float32, device=dev)
    elif return_probs:
        raise ValueError("greedy sampling produces no probabilities")
    need = sample_workspace_bytes(R, V, draws, mode)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        rc = _lib.load().cfa_sample(
            x.data_ptr(), x.stride(0), _KINDS[input_kind], R, V, draws, float(temperature),
            int(top_k), float(top_p), _SMODES[mode], u.data_ptr() if u is not None else None,
            out.data_ptr(), probs.data_ptr() if probs is not None else None,
            workspace.data_ptr(), workspace.numel(), _stream_ptr(dev))
    _lib.check(rc, "cfa_sample")
    return (out, probs) if return_probs else out


def fused_sampling_triton(logits: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """sampling_triton.py:40-66: the argmax of softmax(logits / T) per row
    (the argmax of the logits; first index on ties).  int32 [batch_size]."""
    if logits.dim() != 2:
        raise ValueError("logits must be [batch_size, vocab_size]")
    return sample(logits, mode="greedy")[:, 0].contiguous()


def launch_fused_sampling(params: SamplingParams, stream: Optional[torch.cuda.Stream] = None,
                          uniforms: Optional[torch.Tensor] = None) -> torch.Tensor:
    """sampling.h:195-216.  Writes params.output_tokens (allocated when None)
    and returns it."""
    x = params.logits
    if params.batch_size <= 0 or params.vocab_size <= 0 or x is None:
        raise ValueError("Invalid batch size or vocab size for sampling launch.")
    if x.dim() != 2 or tuple(x.shape) != (params.batch_size, params.vocab_size):
        raise ValueError("logits must be [batch_size, vocab_size]")
    ctx = torch.cuda.stream(stream) if stream is not None else _Null()
    with ctx:
        if params.temperature <= 1e-5:
            tok = sample(x, mode="greedy")[:, 0]
        else:
            gen = None
            if uniforms is None:
                gen = torch.Generator(device=x.device)
                gen.manual_seed(int(params.rng_seed))
            u = None if uniforms is None else uniforms.reshape(-1, 1).float()
            tok = sample(x, mode="multinomial", temperature=params.temperature, uniforms=u,
                         generator=gen)[:, 0]
        if params.output_tokens is None:
            params.output_tokens = torch.empty(params.batch_size, dtype=torch.int32,
                                               device=x.device)
        params.output_tokens.copy_(tok)
    return params.output_tokens


def expand_tree_level(draft_rows: torch.Tensor, *, children: int = 2, mode: str = "sample",
                      temperature: float = 1.0, uniforms: Optional[torch.Tensor] = None,
                      generator: Optional[torch.Generator] = None,
                      return_probs: bool = False):
    """Children of one level of draft-tree nodes: draft_rows [R, V] logits of
    the R nodes; returns int32 [R, children].

    mode "sample": i.i.d. draws from softmax(row / T) -- what multi-candidate
    rejection sampling (cfa_tree_verify, cpp mode) assumes of a node's
    children; "greedy": the `children` most likely tokens (greedy
    verification)."""
    if mode == "sample":
        return sample(draft_rows, mode="multinomial", temperature=temperature, draws=children,
                      uniforms=uniforms, generator=generator, return_probs=return_probs)
    if mode == "greedy":
        out = sample(draft_rows, mode="greedy", draws=children)
        return (out, None) if return_probs else out
    raise ValueError("mode must be 'sample' or 'greedy'")


_ROW_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def sample_rows_workspace_bytes(R: int, V: int) -> int:
    return int(_lib.load().cfa_sample_rows_workspace_size(R, V))


def _setting(name: str, value, R: int, dtype: torch.dtype, dev, ok, says: str):
    """(device pointer or None, scalar, what to keep alive) of a row setting."""
    if isinstance(value, torch.Tensor):
        _require_cuda(name, value, dtype, dev)
        if tuple(value.shape) != (R,):
            raise ValueError(f"{name} must be a number or [R] = [{R}]")
        value = value.contiguous()
        return value.data_ptr(), 0, value
    if not ok(value):
        raise ValueError(f"{name} must be {says}")
    return None, value, None


def sample_rows(rows: torch.Tensor, uniforms: Optional[torch.Tensor] = None, *,
                temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, draws: Optional[int] = None,
                generator: Optional[torch.Generator] = None, return_probs: bool = False,
                workspace: Optional[torch.Tensor] = None):
    """Draw from rows [R, V] of logits (fp32, bf16 or fp16), each row with its
    own settings: temperature, top_p, min_p (fp32 [R] tensors) and top_k (int32
    [R]), or numbers for all rows.

    A row keeps its first tokens in the order of falling logits (equal ones:
    lower index first): rank < top_k (<= 0: off), softmax mass in front < top_p
    (1: off), probability >= min_p times the largest (0: off); temperature 0
    keeps the largest alone.  The three are intersected: top_p is of the whole
    row's mass, not of what top_k left, and keeps no fewer tokens than filters one
    after the other, which renormalise in between.  uniforms fp32 [R, draws] in [0, 1) pick the first
    kept index whose kept mass exceeds u of the whole; without them they come
    from `generator` (`draws` a row, default 1).  -inf masks a token; a row of
    masked tokens alone gives -1.  Returns int32 [R, draws], and with
    return_probs the renormalised probabilities [R, V] fp32 the draws used.
    """
    if not isinstance(rows, torch.Tensor) or rows.device.type != "cuda":
        raise ValueError("rows must be a HIP device tensor")
    if rows.dtype not in _ROW_TYPES:
        raise ValueError("rows must be float32, bfloat16 or float16")
    if rows.dim() != 2 or rows.shape[1] == 0:
        raise ValueError("rows must be [R, V] with V > 0")
    R, V = rows.shape
    dev = rows.device
    if rows.stride(1) != 1 or (R > 1 and rows.stride(0) < V):
        rows = rows.contiguous()
    if uniforms is not None:
        _require_cuda("uniforms", uniforms, torch.float32, dev)
        if uniforms.dim() != 2 or uniforms.shape[0] != R or draws not in (None, uniforms.shape[1]):
            raise ValueError("uniforms must be [R, draws]")
        uniforms = uniforms.contiguous()
        draws = uniforms.shape[1]
    else:
        draws = 1 if draws is None else int(draws)
        if draws < 0:
            raise ValueError("draws must not be negative")
        uniforms = torch.rand(R, draws, device=dev, generator=generator, dtype=torch.float32)
    settings = [
        _setting("temperature", temperature, R, torch.float32, dev,
                 lambda v: 0.0 <= v < float("inf"), "finite and not negative"),
        _setting("top_k", top_k, R, torch.int32, dev, lambda v: v == int(v), "an integer"),
        _setting("top_p", top_p, R, torch.float32, dev, lambda v: 0.0 < v <= 1.0, "in (0, 1]"),
        _setting("min_p", min_p, R, torch.float32, dev, lambda v: 0.0 <= v <= 1.0, "in [0, 1]")]
    (t, t0, _), (k, k0, _), (p, p0, _), (m, m0, _) = settings
    k0 = min(max(int(k0), 0), 2 ** 31 - 1)
    tokens = torch.empty(R, draws, dtype=torch.int32, device=dev)
    probs = torch.empty(R, V, dtype=torch.float32, device=dev) if return_probs else None
    lib = _lib.load()
    need = int(lib.cfa_sample_rows_workspace_size(R, V))
    workspace = _workspace(workspace, need, dev)
    with _on(dev):
        rc = lib.cfa_sample_rows(
            rows.data_ptr(), rows.stride(0), _ROW_TYPES[rows.dtype], R, V, draws, t, t0, k, k0, p,
            p0, m, m0, uniforms.data_ptr(), tokens.data_ptr(),
            probs.data_ptr() if return_probs else None, workspace.data_ptr(), workspace.numel(),
            _stream_ptr(dev))
    _lib.check(rc, "cfa_sample_rows")
    return (tokens, probs) if return_probs else tokens


def filtered_probs(rows: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The probabilities [R, V] fp32 that sample_rows draws from: what
    ``verify.chain_verify`` and ``verify.tree_verify`` take as
    ``input_kind="probs"`` of filtered distributions."""
    return sample_rows(rows, draws=0, temperature=temperature, top_k=top_k, top_p=top_p,
                       min_p=min_p, return_probs=True, workspace=workspace)[1]


def _rows_strides(x: torch.Tensor):
    """(B, N, V, stride of sequences, stride of rows) of [B, V] or [B, N, V]."""
    if x.dim() == 2:
        return x.shape[0], 1, x.shape[1], x.stride(0), x.stride(0)
    return (*x.shape, x.stride(0), x.stride(1))


def _span(x: torch.Tensor):
    """First byte and the one behind the last that x covers."""
    if x.numel() == 0:
        return x.data_ptr(), x.data_ptr()
    last = sum((n - 1) * st for n, st in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def adjust_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None,
                  history_lens: Optional[torch.Tensor] = None,
                  prompt_lens: Optional[torch.Tensor] = None, repetition=1.0, frequency=0.0,
                  presence=0.0, node_tokens: Optional[torch.Tensor] = None,
                  tree_mask: Optional[torch.Tensor] = None,
                  bias_tokens: Optional[torch.Tensor] = None,
                  bias_values: Optional[torch.Tensor] = None,
                  allowed: Optional[torch.Tensor] = None,
                  allowed_index: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None,
                  out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Penalties of repeated tokens, biases and grammar masks on logits [B, V], or
    [B, N, V] (N rows of each sequence: a draft tree's nodes, a chain's places);
    fp32, bf16 or fp16.  Returns them in `out_dtype` (their own, or float32).

    history [B, L] int32 holds each sequence's tokens, history_lens [B] int32 how
    many of them count (default L), prompt_lens [B] int32 how many of those are its
    prompt (default 0).  A token seen anywhere there has its logit divided (if
    positive) or multiplied by `repetition`; one that stands c > 0 times behind the
    prompt loses frequency * c + presence.  The three are numbers, or fp32 [B]
    tensors.  With node_tokens [B, N] int32 and tree_mask (int64 [N] or [B, N], each
    node's ancestor-or-self mask) a row also counts the tokens of its own path, as
    generated ones; N is then at most 64.  (A chain is a tree of one path; a first
    node whose token the history has already goes in as -1.)

    bias_tokens int32 and bias_values fp32, [K] or [B, K], are added to their tokens'
    logits; of the same token twice the last.  Ids outside the vocabulary, here, in
    the history and in node_tokens, are passed over: -1 pads.  allowed int32 [M,
    ceil(V / 32)] holds grammars' masks, token v in bit v % 32 of word v / 32, and
    allowed_index int32 ([B] or [B, N]) the mask of each row (-1: none); without it
    there is one for each row.  Masked tokens get -inf.

    In fp32, rounded once.  out (default a new tensor) may be `logits` itself: what
    nothing changes is then not touched.  Another tensor must not overlap them.
    """
    if not isinstance(logits, torch.Tensor) or logits.device.type != "cuda":
        raise ValueError("logits must be a HIP device tensor")
    if logits.dtype not in _ROW_TYPES:
        raise ValueError("logits must be float32, bfloat16 or float16")
    if logits.dim() not in (2, 3) or logits.shape[-1] == 0:
        raise ValueError("logits must be [B, V] or [B, N, V] with V > 0")
    dev = logits.device
    inplace = out is logits
    if logits.stride(-1) != 1 and not inplace:
        logits = logits.contiguous()
    B, N, V, sb, sn = _rows_strides(logits)

    def ints(name, t, shape):
        if t is None:
            return None
        _require_cuda(name, t, torch.int32, dev)
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must be {list(shape)}")
        return t.contiguous()

    if history is None and (history_lens is not None or prompt_lens is not None):
        raise ValueError("history_lens and prompt_lens go with history")
    if history is not None:
        _require_cuda("history", history, torch.int32, dev)
        if history.dim() != 2 or history.shape[0] != B:
            raise ValueError(f"history must be [B, L] with B = {B}")
        history = history.contiguous()
    L = 0 if history is None else history.shape[1]
    history_lens = ints("history_lens", history_lens, (B,))
    prompt_lens = ints("prompt_lens", prompt_lens, (B,))
    settings = [
        _setting("repetition", repetition, B, torch.float32, dev,
                 lambda v: 0.0 < v < float("inf"), "finite and positive"),
        _setting("frequency", frequency, B, torch.float32, dev,
                 lambda v: abs(v) < float("inf"), "finite"),
        _setting("presence", presence, B, torch.float32, dev,
                 lambda v: abs(v) < float("inf"), "finite")]
    (r, r0, _), (f, f0, _), (p, p0, _) = settings
    if (node_tokens is None) != (tree_mask is None):
        raise ValueError("node_tokens and tree_mask go together")
    mstride = 0
    if node_tokens is not None:
        if logits.dim() != 3 or N > 64:
            raise ValueError("node_tokens go with logits [B, N, V] of at most 64 nodes")
        node_tokens = ints("node_tokens", node_tokens, (B, N))
        _require_cuda("tree_mask", tree_mask, torch.int64, dev)
        if tuple(tree_mask.shape) == (B, N):
            mstride = N
        elif tuple(tree_mask.shape) != (N,):
            raise ValueError("tree_mask must be [N] or [B, N]")
        tree_mask = tree_mask.contiguous()
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values go together")
    K = bstride = 0
    if bias_tokens is not None:
        _require_cuda("bias_tokens", bias_tokens, torch.int32, dev)
        _require_cuda("bias_values", bias_values, torch.float32, dev)
        if bias_tokens.shape != bias_values.shape or bias_tokens.dim() not in (1, 2) or (
                bias_tokens.dim() == 2 and bias_tokens.shape[0] != B):
            raise ValueError("bias_tokens and bias_values must both be [K] or [B, K]")
        K = bias_tokens.shape[-1]
        bstride = K if bias_tokens.dim() == 2 else 0
        bias_tokens, bias_values = bias_tokens.contiguous(), bias_values.contiguous()
    words = masks = 0
    if allowed is None and allowed_index is not None:
        raise ValueError("allowed_index goes with allowed")
    if allowed is not None:
        _require_cuda("allowed", allowed, torch.int32, dev)
        words = (V + 31) // 32
        rows = tuple(logits.shape[:-1])
        if allowed_index is not None:
            allowed_index = ints("allowed_index", allowed_index, rows)
            if allowed.dim() != 2 or allowed.shape[1] != words:
                raise ValueError(f"allowed must be [M, ceil(V / 32)] = [M, {words}]")
        elif tuple(allowed.shape) not in ((*rows, words), (B * N, words)):
            raise ValueError("without allowed_index, allowed must have a mask for each row")
        allowed = allowed.contiguous()
        masks = allowed.numel() // words
    if out is None:
        out_dtype = logits.dtype if out_dtype is None else out_dtype
        if out_dtype not in (logits.dtype, torch.float32):
            raise ValueError("out_dtype must be float32 or the logits' dtype")
        out = torch.empty(logits.shape, dtype=out_dtype, device=dev)
    else:
        if not isinstance(out, torch.Tensor) or out.dtype not in (logits.dtype, torch.float32) or (
                out_dtype not in (None, out.dtype)):
            raise ValueError("out must be float32 or of the logits' dtype (and of out_dtype)")
        _require_cuda("out", out, out.dtype, dev)
        if out.shape != logits.shape or out.stride(-1) != 1:
            raise ValueError("out must have the logits' shape and a contiguous last dimension")
        _, _, _, ob, on = _rows_strides(out)
        if (N > 1 and on < V) or (B > 1 and ob < (N - 1) * on + V):
            raise ValueError("out's rows must not overlap")
        same = (out.data_ptr() == logits.data_ptr() and out.dtype == logits.dtype
                and out.stride() == logits.stride())
        (lo, hi), (olo, ohi) = _span(logits), _span(out)
        if not same and lo < ohi and olo < hi:
            raise ValueError("out must be the logits themselves or not overlap them")
    _, _, _, ob, on = _rows_strides(out)
    with _on(dev):
        rc = _lib.load().cfa_adjust_logits(
            logits.data_ptr(), sb, sn, _ROW_TYPES[logits.dtype], B, N, V, _ptr(history),
            _ptr(history_lens), _ptr(prompt_lens), L, r, r0, f, f0, p, p0, _ptr(node_tokens),
            _ptr(tree_mask), mstride, _ptr(bias_tokens), _ptr(bias_values), bstride, K,
            _ptr(allowed), words, masks, _ptr(allowed_index), out.data_ptr(), ob, on,
            out.dtype == torch.float32, _stream_ptr(dev))
    _lib.check(rc, "cfa_adjust_logits")
    return out


class _Null:
    def __enter__(self):
        return self

    def __exit__(self, *a):
        return False
