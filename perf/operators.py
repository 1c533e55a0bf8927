"""Workloads of the attention side of a decoder layer and of the sampler behind
it, for decoders that normalise their heads, scale their rotations, cap or bias
their scores, or filter their draws for each request.

A case is a dict of plain values; ``kind`` names its operator:

  rope    ``rotary.qk_norm_rope_kv``: RMSNorm of every q and k head, rotary
          positions and the write of k and v into the paged cache, in one pass
  tree    ``verify.tree_attention`` with a tanh cap, a distance bias or a
          sliding window: draft trees, and single tokens (a tree of one node)
  prompt  ``verify.prompt_attention``: chunks of prompts of different lengths,
          causal over the paged cache, with the same scores
  sample  ``sampling.sample_rows``: temperature, top-k, top-p and min-p of
          each row's own, from given uniforms

``run`` computes them in elementary torch operations, or, where ``own`` is
true, makes the package's calls.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16


def listed():
    return [
        # one decode step of a small batch far along its conversations
        dict(name="rope_decode_b8", kind="rope", lens="1 " * 8, ctx=40, pos0=100000, Hq=32, Hkv=8,
             D=128, rot=128, layout="half", scaling="bands", norm=True, dtype="bfloat16", pad=0),
        # the benchmark's verify step: 8 sequences x 63 nodes, part of the head rotated
        dict(name="rope_verify_m504", kind="rope", lens="63 " * 8, ctx=2048, pos0=0, Hq=32, Hkv=8,
             D=128, rot=64, layout="interleaved", scaling="none", norm=True, dtype="bfloat16",
             pad=0),
        # a step's prompt chunks, packed and padded at the end
        dict(name="rope_prompt_8k", kind="rope", lens="4111 37 1 2600 1400", ctx=129, pos0=0,
             Hq=32, Hkv=8, D=128, rot=128, layout="half", scaling="yarn", norm=True,
             dtype="bfloat16", pad=43),
        # plain decode of one user behind a sliding window, biased by distance
        dict(name="decode_b1_window", kind="tree", B=1, N=1, Hq=32, Hkv=8, D=128, ctx=1500,
             ragged=False, cap=0.0, alibi=True, window=1024, dtype="bfloat16"),
        # plain decode of a full batch at the benchmark's context, capped scores
        dict(name="decode_b64_cap", kind="tree", B=64, N=1, Hq=32, Hkv=8, D=128, ctx=4096,
             ragged=True, cap=50.0, alibi=False, window=0, dtype="bfloat16"),
        # a few users' small trees at the draft's heads, biased by distance
        dict(name="tree_b3_alibi", kind="tree", B=3, N=31, Hq=32, Hkv=8, D=64, ctx=1500,
             ragged=True, cap=0.0, alibi=True, window=0, dtype="float16"),
        # the benchmark's verification step with capped scores
        dict(name="tree_b16_cap", kind="tree", B=16, N=63, Hq=32, Hkv=8, D=128, ctx=4096,
             ragged=False, cap=50.0, alibi=False, window=0, dtype="bfloat16"),
        # short prompts joining a step, the rest of one behind its first chunk
        dict(name="prompt_ragged", kind="prompt", lens="311 1 700 64 17", ctx="0 900 512 0 77",
             Hq=32, Hkv=8, D=64, cap=0.0, alibi=True, window=500, dtype="float16", pad=3),
        # one long prompt with capped scores
        dict(name="prompt_8k_cap", kind="prompt", lens="8192", ctx="0", Hq=32, Hkv=8, D=128,
             cap=50.0, alibi=False, window=0, dtype="bfloat16", pad=0),
        # one user's next token at the small test models' vocabulary
        dict(name="sample_r1", kind="sample", R=1, V=32000, draws=1, probs=False,
             dtype="float32", mix=False),
        # a step's requests, each with its own settings, from bf16 logits
        dict(name="sample_r64_mixed", kind="sample", R=64, V=128256, draws=1, probs=False,
             dtype="bfloat16", mix=True),
        # the filtered rows of a verification: 8 sequences x 9 positions
        dict(name="sample_r72_probs", kind="sample", R=72, V=128256, draws=1, probs=True,
             dtype="float32", mix=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(values):
    return " ".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split()]


def draw(rng):
    kind = rng.choice(["rope", "tree", "prompt", "sample"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    D = rng.choice([128, 128, 64])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (16, 16), (16, 8), (8, 1)])
    if kind == "rope":
        lens = [_log_int(rng, 1, 1600) for _ in range(rng.randint(1, 5))]
        if rng.random() < 0.4:
            lens = [rng.choice([1, 1, 7, 31, 63])] * _log_int(rng, 1, 64)
        return dict(kind=kind, lens=_text(lens), ctx=_log_int(rng, 1, 2048),
                    pos0=rng.choice([0, 0, 31000, 100000]), Hq=Hq, Hkv=Hkv, D=D,
                    rot=rng.choice([D, D, D // 2, D // 4]),
                    layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "bands", "yarn"]),
                    norm=rng.choice([True, True, False]), dtype=dtype, pad=rng.choice([0, 0, 5]))
    cap = rng.choice([0.0, 30.0, 50.0])
    alibi = rng.choice([True, False]) if cap else rng.choice([True, True, False])
    window = rng.choice([0, 0, _log_int(rng, 1, 2048)])
    if not cap and not alibi and not window:
        window = _log_int(rng, 1, 2048)
    if kind == "tree":
        N = rng.choice([1, 1, rng.randint(2, 63)])
        return dict(kind=kind, B=_log_int(rng, 1, 64 if N == 1 else 16), N=min(N, 256 * Hkv // Hq),
                    Hq=Hq, Hkv=Hkv, D=D, ctx=_log_int(rng, 64, 4096),
                    ragged=rng.choice([True, False]), cap=cap, alibi=alibi, window=window,
                    dtype=dtype)
    if kind == "prompt":
        n = rng.randint(1, 6)
        return dict(kind=kind, lens=_text(_log_int(rng, 1, 2600) for _ in range(n)),
                    ctx=_text(rng.choice([0, 0, _log_int(rng, 1, 2048)]) for _ in range(n)), Hq=Hq,
                    Hkv=Hkv, D=D, cap=cap, alibi=alibi, window=window, dtype=dtype,
                    pad=rng.choice([0, 0, 5]))
    return dict(kind=kind, R=_log_int(rng, 1, 64), V=_log_int(rng, 8000, 128256),
                draws=rng.choice([1, 1, 2]), probs=rng.choice([True, False]),
                dtype=rng.choice(["float32", "bfloat16", "float16"]),
                mix=rng.choice([True, True, False]))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    return _PREPARE[case["kind"]](case, _gen(seed))


def run(state):
    return _RUN[state["case"]["kind"]](state)


def work(case):
    return _WORK[case["kind"]](case)


def exact(case, seed):
    return _EXACT[case["kind"]](case, prepare(case, seed))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(slots, g):
    """Block tables [B, pages] int32 over one pool for sequences of `slots`
    slots, and the pool's number of blocks; -1 behind a sequence's last page."""
    need = [(n + PAGE - 1) // PAGE for n in slots]
    nblk = sum(need) + 5
    perm = torch.randperm(nblk, device="cuda", generator=g).int()
    tables = torch.full((len(slots), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = perm[at: at + n]
        at += n
    return tables, nblk


def _pools(case, nblk, g):
    shape = (nblk, 1, case["Hkv"], PAGE, case["D"])
    dt = getattr(torch, case["dtype"])
    return (torch.randn(shape, device="cuda", generator=g).to(dt),
            torch.randn(shape, device="cuda", generator=g).to(dt))


# -- rotary positions with head norms and the cache write ------------------------

THETA = 500000.0
SCALINGS = {
    "none": None,
    "linear": dict(kind="linear", factor=4.0),
    "ntk": dict(kind="ntk", factor=4.0),
    "bands": dict(kind="bands", factor=8.0, low=1.0, high=4.0, original=8192),
    "yarn": dict(kind="yarn", factor=16.0, original=4096),
}


def _prepare_rope(case, g):
    lens, ctx, Hq, Hkv, D = _ints(case["lens"]), *(case[k] for k in ("ctx", "Hq", "Hkv", "D"))
    dt = getattr(torch, case["dtype"])
    B, T = len(lens), sum(lens) + case["pad"]
    base = [max(1, ctx - 5 * b) for b in range(B)]
    tables, nblk = _tables([c + n for c, n in zip(base, lens)], g)
    kp, vp = _pools(case, nblk, g)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, device="cuda", generator=g).to(dt)
    cu = np.concatenate([[0], np.cumsum(lens)])
    pos = np.zeros(T, np.int64)
    for b in range(B):
        pos[cu[b]: cu[b + 1]] = case["pos0"] + base[b] + np.arange(lens[b])
    norms = [(1.0 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dt) for _ in range(2)]
    s = dict(case=case, qkv=qkv, pos=_int32(pos.tolist()), cu=_int32(cu.tolist()), cu_host=cu,
             base=_int32(base), base_host=base, tables=tables, kp=kp, vp=vp,
             norms=norms if case["norm"] else [None, None],
             q_out=torch.zeros(T, Hq, D, dtype=dt, device="cuda"))
    if own:
        from cudaforge_amd.rotary import Rotary

        s["rotary"] = Rotary(case["rot"], THETA, layout=case["layout"],
                             scaling=SCALINGS[case["scaling"]], device="cuda")
    return s


def _heads(s):
    case = s["case"]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    x = s["qkv"].view(-1, Hq + 2 * Hkv, D)
    return x[:, :Hq], x[:, Hq: Hq + Hkv], x[:, Hq + Hkv:]


def _frequencies(case):
    """Radians per position of each rotated pair, and the factor on the rotation."""
    rot, sc = case["rot"], SCALINGS[case["scaling"]]
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    kind = sc["kind"] if sc else "none"
    theta = THETA * sc["factor"] ** (rot / (rot - 2)) if kind == "ntk" else THETA
    inv = theta ** (-i / rot)
    if kind == "linear":
        inv = inv / sc["factor"]
    elif kind == "bands":
        turns = sc["original"] * inv / (2 * math.pi)      # turns over the trained length
        mix = ((turns - sc["low"]) / (sc["high"] - sc["low"])).clamp(0.0, 1.0)
        inv = inv * (mix + (1.0 - mix) / sc["factor"])
    elif kind == "yarn":
        def at(beta):
            return rot * math.log(sc["original"] / (beta * 2 * math.pi)) / (2 * math.log(THETA))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        inv = inv * (1.0 - ramp) + inv / sc["factor"] * ramp
        return inv, 0.1 * math.log(sc["factor"]) + 1.0
    return inv, 1.0


EPS = 1e-6


def _run_rope(s):
    case = s["case"]
    q, k, v = _heads(s)
    if own:
        from cudaforge_amd.rotary import qk_norm_rope_kv

        # sequences of one length need no table of where each begins
        uniform = len(set(_ints(case["lens"]))) == 1 and not case["pad"]
        out = qk_norm_rope_kv(
            q, k, v, s["pos"], s["rotary"], s["kp"], s["vp"], s["tables"], s["base"],
            cu_seqlens=None if uniform else s["cu"], q_norm=s["norms"][0], k_norm=s["norms"][1],
            eps=EPS, q_out=s["q_out"])
        return dict(q=out, keys=s["kp"], values=s["vp"])
    n, rot = int(s["cu_host"][-1]), case["rot"]
    inv, factor = _frequencies(case)
    ang = s["pos"][:n].double()[:, None] * inv
    cos = (ang.cos() * factor).float()[:, None, :]
    sin = (ang.sin() * factor).float()[:, None, :]

    def turned(x, w):
        x = x[:n].float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        r, rest = x[..., :rot], x[..., rot:]
        if case["layout"] == "half":
            a, b = r[..., : rot // 2], r[..., rot // 2:]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([r, rest], -1).to(s["q_out"].dtype)

    s["q_out"][:n] = turned(q, s["norms"][0])
    kr = turned(k, s["norms"][1])
    seq = torch.repeat_interleave(torch.arange(len(s["base_host"]), device="cuda"),
                                  (s["cu"][1:] - s["cu"][:-1]).long(), output_size=n)
    slot = s["base"].long()[seq] + torch.arange(n, device="cuda") - s["cu"].long()[seq]
    block = s["tables"][seq, slot // PAGE].long()
    s["kp"][block, 0, :, slot % PAGE] = kr
    s["vp"][block, 0, :, slot % PAGE] = v[:n]
    return dict(q=s["q_out"], keys=s["kp"], values=s["vp"])


def _work_rope(case):
    T, D = sum(_ints(case["lens"])), case["D"]
    heads = case["Hq"] + 2 * case["Hkv"]
    return {"bytes": 2 * 2 * T * heads * D, "flops": 10 * T * (case["Hq"] + case["Hkv"]) * D}


def _exact_rope(case, s):
    n, rot, lay = int(s["cu_host"][-1]), case["rot"], case["layout"]
    inv, factor = _frequencies(case)
    pos = s["pos"][:n].double()
    # each pair as a complex number turned by its angle
    turn = torch.polar(torch.full((n, rot // 2), factor, dtype=torch.float64, device="cuda"),
                       torch.outer(pos, inv)).unsqueeze(1)
    out = []
    for x, w in zip(_heads(s), s["norms"] + ["v"]):
        y = x[:n].double()
        if w is not None and not isinstance(w, str):
            y = y / (y.pow(2).sum(-1, keepdim=True) / case["D"] + EPS).sqrt() * w.double()
        if not isinstance(w, str):
            i = torch.arange(rot // 2, device="cuda")
            a, b = (i, i + rot // 2) if lay == "half" else (2 * i, 2 * i + 1)
            z = torch.complex(y[..., a], y[..., b]) * turn
            y = y.clone()
            y[..., a], y[..., b] = z.real, z.imag
        out.append(y)
    q = s["q_out"].double()
    q[:n] = out[0]
    kp, vp = s["kp"].double(), s["vp"].double()
    tables = s["tables"].tolist()
    for b, m in enumerate(_ints(case["lens"])):
        t0 = int(s["cu_host"][b])
        j = 0
        while j < m:                                    # page by page
            slot = s["base_host"][b] + j
            cnt = min(m - j, PAGE - slot % PAGE)
            blk, o = tables[b][slot // PAGE], slot % PAGE
            kp[blk, 0, :, o: o + cnt] = out[1][t0 + j: t0 + j + cnt].transpose(0, 1)
            vp[blk, 0, :, o: o + cnt] = out[2][t0 + j: t0 + j + cnt].transpose(0, 1)
            j += cnt
    return dict(q=q, keys=kp, values=vp)


# -- attention with capped or biased scores ------------------------------------

def _slopes(case):
    """Geometric slopes 2^(-8 (h + 1) / Hq) of the distance bias, fp32 [Hq]."""
    H = case["Hq"]
    h = torch.arange(1, H + 1, dtype=torch.float64, device="cuda")
    return (2.0 ** (-8.0 * h / H)).float()


def _ancestors(N):
    """[N] int: bit j of entry i says that node j is i or above it, in the
    complete binary tree numbered level by level."""
    masks = []
    for i in range(N):
        masks.append((masks[(i - 1) // 2] if i else 0) | (1 << i))
    return masks


def _tree_lens(case, g):
    B, ctx = case["B"], case["ctx"]
    lens = torch.full((B,), ctx, dtype=torch.int32, device="cuda")
    if case["ragged"] and B > 1:
        lens = torch.randint(max(1, ctx // 4), ctx + 1, (B,), device="cuda", generator=g).int()
        lens[0] = ctx
    return lens


def _score_args(case):
    return dict(soft_cap=case["cap"], alibi_slopes=_slopes(case) if case["alibi"] else None,
                window=case["window"])


def _prepare_tree(case, g):
    B, N, Hq, D = (case[k] for k in ("B", "N", "Hq", "D"))
    lens = _tree_lens(case, g)
    host = lens.tolist()
    tables, nblk = _tables([n + N for n in host], g)
    kp, vp = _pools(case, nblk, g)
    q = (torch.randn(B, N, Hq, D, device="cuda", generator=g) * 2.0).to(kp.dtype)
    masks = torch.tensor(np.array(_ancestors(N), dtype=np.uint64).view(np.int64), device="cuda")
    return dict(case=case, q=q, kp=kp, vp=vp, tables=tables, lens=lens, host=host, masks=masks,
                max_keys=case["ctx"] + N, score=_score_args(case))


def _rows(pool, table, n):
    """The first n slots of a sequence: [Hkv, n, D]."""
    x = pool[table[: (n + PAGE - 1) // PAGE].long(), 0]
    return x.transpose(0, 1).reshape(pool.shape[2], -1, pool.shape[4])[:, :n]


def _attend(case, score, q, k, v, dist, see):
    """q [n, Hq, D], k / v [Hkv, S, D], dist [n, S] = how far each key lies
    behind each query, see [n, S]: what the mask leaves; fp32 [n, Hq, D]."""
    n, Hq, D = q.shape
    Hkv, S, _ = k.shape
    G = Hq // Hkv
    if case["window"]:
        see = see & (dist < case["window"])
    qh = q.float().transpose(0, 1).reshape(Hkv, G, n, D)
    kh, vh = k.float().transpose(1, 2).contiguous(), v.float().contiguous()
    out = torch.empty(Hkv, G, n, D, device="cuda")
    step = max(1, min(Hkv, 2 ** 29 // (G * n * S)))       # KV heads at a time
    for h in range(0, Hkv, step):
        e = min(Hkv, h + step)
        sc = (qh[h:e].reshape(e - h, G * n, D) @ kh[h:e]).view(e - h, G, n, S) * (D ** -0.5)
        if case["cap"]:
            sc = torch.tanh(sc / case["cap"]) * case["cap"]
        if case["alibi"]:
            sc = sc - score["alibi_slopes"].view(Hkv, G, 1, 1)[h:e] * dist
        sc = torch.where(see, sc, float("-inf"))
        top = sc.max(-1, keepdim=True).values
        p = torch.exp(sc - torch.where(top > float("-inf"), top, 0.0))
        total = p.sum(-1, keepdim=True)
        o = (p.view(e - h, G * n, S) @ vh[h:e]).view(e - h, G, n, D)
        out[h:e] = o / torch.where(total > 0, total, 1.0)
    return out.view(Hq, n, D).transpose(0, 1)


def _run_tree(s):
    case = s["case"]
    if own:
        from cudaforge_amd.verify import tree_attention

        return tree_attention(s["q"], s["kp"], s["vp"], s["tables"], s["lens"], s["masks"],
                              max_keys=s["max_keys"], **s["score"])
    N = case["N"]
    bits = (s["masks"][:, None] >> torch.arange(N, device="cuda")) & 1
    depth = bits.sum(-1) - 1
    out = torch.empty_like(s["q"])
    for b, ctx in enumerate(s["host"]):
        at = torch.cat([torch.arange(ctx, device="cuda"), ctx + depth])
        see = torch.cat([torch.ones(N, ctx, dtype=torch.bool, device="cuda"), bits.bool()], 1)
        dist = (ctx + depth)[:, None] - at
        out[b] = _attend(case, s["score"], s["q"][b], _rows(s["kp"], s["tables"][b], ctx + N),
                         _rows(s["vp"], s["tables"][b], ctx + N), dist, see).to(out.dtype)
    return out


def _attention_work(case, queries, pairs, keys):
    D = case["D"]
    return {"bytes": 4 * case["Hkv"] * keys * D + 4 * queries * case["Hq"] * D,
            "flops": 4 * case["Hq"] * D * pairs}


def _work_tree(case):
    B, N, W = case["B"], case["N"], case["window"]
    depths = [bin(m).count("1") - 1 for m in _ancestors(N)]
    lens = [case["ctx"]] * B
    if case["ragged"] and B > 1:
        lens[1:] = [int(0.625 * case["ctx"])] * (B - 1)
    pairs = keys = 0
    for ctx in lens:
        own_path = [d + 1 if not W else min(d + 1, W) for d in depths]
        behind = [ctx if not W else max(0, min(ctx, W - 1 - d)) for d in depths]
        pairs += sum(own_path) + sum(behind)
        keys += max(behind) + N
    return _attention_work(case, B * N, pairs, keys)


def _attend64(case, q, k, v, dist, see):
    """The same in fp64, a few hundred queries at a time, from the shares
    exp(score) / sum of them."""
    n, Hq, D = q.shape
    G = Hq // k.shape[0]
    slope = _slopes(case).double()
    out = torch.zeros(n, Hq, D, dtype=torch.float64, device="cuda")
    for lo in range(0, n, 512):
        rows = slice(lo, min(n, lo + 512))
        hidden = ~see[rows]
        if case["window"]:
            hidden = hidden | (dist[rows] >= case["window"])
        for h in range(Hq):
            sc = torch.mm(q[rows, h].double(), k[h // G].double().t()) / math.sqrt(D)
            if case["cap"] > 0:
                e = torch.exp(-2.0 * sc.abs() / case["cap"])
                sc = case["cap"] * sc.sign() * (1.0 - e) / (1.0 + e)
            if case["alibi"]:
                sc = sc - slope[h] * dist[rows].double()
            share = torch.softmax(sc.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
            out[rows, h] = torch.mm(share, v[h // G].double())
    return out


def _exact_tree(case, s):
    N, B = case["N"], case["B"]
    anc = _ancestors(N)
    tree = torch.tensor([[(m >> j) & 1 == 1 for j in range(N)] for m in anc], device="cuda")
    depth = torch.tensor([bin(m).count("1") - 1 for m in anc], device="cuda")
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(B):
        ctx = s["host"][b]
        see = torch.ones(N, ctx + N, dtype=torch.bool, device="cuda")
        see[:, ctx:] = tree
        far = torch.empty(N, ctx + N, dtype=torch.int64, device="cuda")
        far[:, :ctx] = ctx + depth[:, None] - torch.arange(ctx, device="cuda")
        far[:, ctx:] = depth[:, None] - depth
        out[b] = _attend64(case, s["q"][b], _rows(s["kp"], s["tables"][b], ctx + N),
                           _rows(s["vp"], s["tables"][b], ctx + N), far, see)
    return out


def _prepare_prompt(case, g):
    lens, ctx, Hq, D = _ints(case["lens"]), _ints(case["ctx"]), case["Hq"], case["D"]
    tables, nblk = _tables([c + n for c, n in zip(ctx, lens)], g)
    kp, vp = _pools(case, nblk, g)
    T = sum(lens) + case["pad"]
    q = (torch.randn(T, Hq, D, device="cuda", generator=g) * 2.0).to(kp.dtype)
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    return dict(case=case, q=q, kp=kp, vp=vp, tables=tables, ctx=_int32(ctx), cu=_int32(cu),
                cu_host=cu, max_keys=max(c + n for c, n in zip(ctx, lens)),
                max_query=max(lens), out=torch.zeros_like(q), score=_score_args(case))


def _run_prompt(s):
    case = s["case"]
    if own:
        from cudaforge_amd.verify import prompt_attention

        return prompt_attention(s["q"], s["kp"], s["vp"], s["tables"], s["ctx"], s["cu"],
                                max_query=s["max_query"], max_keys=s["max_keys"], out=s["out"],
                                **s["score"])
    for b, (n, ctx) in enumerate(zip(_ints(case["lens"]), _ints(case["ctx"]))):
        rows = slice(s["cu_host"][b], s["cu_host"][b + 1])
        at = torch.arange(ctx + n, device="cuda")
        dist = at[ctx:, None] - at
        s["out"][rows] = _attend(case, s["score"], s["q"][rows],
                                 _rows(s["kp"], s["tables"][b], ctx + n),
                                 _rows(s["vp"], s["tables"][b], ctx + n), dist,
                                 dist >= 0).to(s["out"].dtype)
    return s["out"]


def _work_prompt(case):
    pairs = keys = 0
    W = case["window"]
    for n, ctx in zip(_ints(case["lens"]), _ints(case["ctx"])):
        seen = [min(ctx + i + 1, W) if W else ctx + i + 1 for i in range(n)]
        pairs += sum(seen)
        keys += min(ctx + n, n + W - 1) if W else ctx + n
    return _attention_work(case, sum(_ints(case["lens"])), pairs, keys)


def _exact_prompt(case, s):
    out = s["out"].double()
    for b, (n, ctx) in enumerate(zip(_ints(case["lens"]), _ints(case["ctx"]))):
        t0 = s["cu_host"][b]
        key = torch.arange(ctx + n, device="cuda")
        far = ctx + key[:n].unsqueeze(1) - key
        out[t0: t0 + n] = _attend64(case, s["q"][t0: t0 + n],
                                    _rows(s["kp"], s["tables"][b], ctx + n),
                                    _rows(s["vp"], s["tables"][b], ctx + n), far, far >= 0)
    return out


# -- sampling --------------------------------------------------------------------

def _prepare_sample(case, g):
    R, V = case["R"], case["V"]
    x = torch.randn(R, V, device="cuda", generator=g) * 2.0
    # tokens that the request's grammar or stop list forbids
    x[torch.rand(R, V, device="cuda", generator=g) < 0.02] = float("-inf")
    s = dict(case=case, rows=x.to(getattr(torch, case["dtype"])),
             u=torch.rand(R, case["draws"], device="cuda", generator=g))
    if case["mix"]:
        def pick(values, dtype=torch.float32):
            at = torch.randint(0, len(values), (R,), device="cuda", generator=g)
            return torch.tensor(values, dtype=dtype, device="cuda")[at]
        s.update(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.3]),
                 top_k=pick([0, 0, 20, 50, 1000], torch.int32),
                 top_p=pick([1.0, 0.8, 0.9, 0.95]), min_p=pick([0.0, 0.0, 0.02, 0.1]))
    else:
        s.update(temperature=0.7, top_k=50, top_p=0.9, min_p=0.05)
    return s


def _settings(s):
    """Each row's temperature, top_k, top_p and min_p as [R, 1] tensors."""
    R = s["case"]["R"]
    out = []
    for key, dt in (("temperature", torch.float32), ("top_k", torch.int64),
                    ("top_p", torch.float32), ("min_p", torch.float32)):
        v = s[key]
        v = v if isinstance(v, torch.Tensor) else torch.full((R,), v, device="cuda")
        out.append(v.to(dt).view(R, 1))
    return out


def _run_sample(s):
    case = s["case"]
    if own:
        from cudaforge_amd.sampling import sample_rows

        res = sample_rows(s["rows"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                          top_p=s["top_p"], min_p=s["min_p"], return_probs=case["probs"])
        return dict(tokens=res[0], probs=res[1]) if case["probs"] else dict(tokens=res)
    # in 64 bits: values next to a border decide whole numbers
    t, k, p, m = (v.double() for v in _settings(s))
    V = case["V"]
    x = s["rows"].double()
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((order.values - order.values[:, :1]) / torch.where(t > 0, t, 1.0))
    before = torch.cumsum(w, -1) - w
    total = w.sum(-1, keepdim=True)
    rank = torch.arange(V, device="cuda")
    k = torch.where(t > 0, torch.where(k > 0, k, float(V)), 1.0)
    keep = (rank < k) & ((before < p * total) | (p >= 1.0)) & (w >= m) & (w > 0)
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, order.indices, torch.where(keep, w, 0.0))
    upto = torch.cumsum(kept, -1)
    tokens = (upto[:, None, :] <= s["u"].double()[:, :, None] * upto[:, None, -1:]).sum(-1)
    last = (kept > 0).long().mul(rank).max(-1, keepdim=True).values
    out = dict(tokens=torch.minimum(tokens, last).int())
    if case["probs"]:
        out["probs"] = (kept / upto[:, -1:]).float()
    return out


def _work_sample(case):
    n = case["R"] * case["V"]
    size = 4 if case["dtype"] == "float32" else 2
    return {"bytes": size * n + (4 * n if case["probs"] else 0) + 8 * case["R"] * case["draws"],
            "flops": 4 * n}


def _exact_sample(case, s):
    """Row by row on the host, from the kept set's own definition."""
    rows = s["rows"].double().cpu().numpy()
    us = s["u"].double().cpu().numpy()
    sets = [v.cpu().numpy().reshape(-1) for v in _settings(s)]
    tokens = np.zeros((case["R"], case["draws"]), np.int32)
    probs = np.zeros(rows.shape) if case["probs"] else None
    for r, x in enumerate(rows):
        t, k, p, m = (float(v[r]) for v in sets)
        if t <= 0:
            kept = np.array([int(np.argmax(x))])
            weight = np.ones(1)
        else:
            by = np.argsort(-x, kind="stable")
            by = by[: int(np.isfinite(x).sum())]
            w = np.exp((x[by] - x[by[0]]) / t)
            n = len(by)
            if p < 1.0:
                n = min(n, 1 + int(np.searchsorted(np.cumsum(w)[:-1], p * w.sum(), side="left")))
            if k > 0:
                n = min(n, int(k))
            if m > 0:
                n = min(n, max(1, int((w >= m).sum())))
            kept = np.sort(by[:n])
            weight = np.exp((x[kept] - x[by[0]]) / t)
        upto = np.cumsum(weight)
        at = np.searchsorted(upto, us[r] * upto[-1], side="right")
        tokens[r] = kept[np.minimum(at, len(kept) - 1)]
        if probs is not None:
            probs[r, kept] = weight / upto[-1]
    out = dict(tokens=torch.from_numpy(tokens).cuda())
    if probs is not None:
        out["probs"] = torch.from_numpy(probs).cuda()
    return out


_PREPARE = {"rope": _prepare_rope, "tree": _prepare_tree, "prompt": _prepare_prompt,
            "sample": _prepare_sample}
_RUN = {"rope": _run_rope, "tree": _run_tree, "prompt": _run_prompt, "sample": _run_sample}
_WORK = {"rope": _work_rope, "tree": _work_tree, "prompt": _work_prompt, "sample": _work_sample}
_EXACT = {"rope": _exact_rope, "tree": _exact_tree, "prompt": _exact_prompt,
          "sample": _exact_sample}
