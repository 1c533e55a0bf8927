"""Workloads of a decoder that keeps its paged cache in 8 bits, looks at long
conversations through a window with a few first tokens beside it, and shapes
the logits in front of its sampler and its verification.

A case is a dict of plain values; ``kind`` names its operator:

  write   ``rotary.qk_norm_rope_kv`` into e4m3 pages with a power-of-two scale
          for each token and head, and ``verify.kv_gather`` of what it wrote
  read    ``verify.kv_gather``: sequences' keys and values out of such pages
  tree    ``verify.tree_attention`` over them, or over 16-bit pages, with a
          sliding window and first tokens that stay visible: draft trees, and
          single tokens (a tree of one node)
  prompt  ``verify.prompt_attention`` of prompt chunks, the same way
  logits  ``sampling.adjust_logits``: penalties of repeated tokens, biases and
          grammar masks, of single rows and of a draft tree's nodes

``run`` computes them in elementary torch operations, or, where ``own`` is
true, makes the package's calls.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16
THETA = 500000.0
EPS = 1e-6
TOP = 448.0          # the largest e4m3 value


def listed():
    return [
        # one decode step of a small batch far along its conversations
        dict(name="write_decode_b8", kind="write", lens="1 " * 8, ctx=40, pos0=100000, Hq=32,
             Hkv=8, D=128, layout="half", norm=True, dtype="bfloat16", pad=0),
        # a step's prompt chunks, packed and padded at the end
        dict(name="write_prompt_8k", kind="write", lens="4111 37 1 2600 1400", ctx=129, pos0=0,
             Hq=32, Hkv=8, D=128, layout="half", norm=True, dtype="bfloat16", pad=43),
        # the last tokens of three conversations, for a layer that keeps no pages
        dict(name="read_b3_tail", kind="read", lens="64 1 300", starts="1000 1699 77", Hkv=8, D=64,
             dtype="float16", pad=0),
        # a full batch's contexts, handed over whole
        dict(name="read_b8_4k", kind="read", lens="4096 " * 8, starts="0 " * 8, Hkv=8, D=128,
             dtype="bfloat16", pad=0),
        # plain decode of one user, a window and four first tokens of a long conversation
        dict(name="decode_b1_sinks", kind="tree", B=1, N=1, Hq=32, Hkv=8, D=128, ctx=30000,
             ragged=False, e4m3=True, window=1024, sinks=4, cap=0.0, dtype="bfloat16"),
        # plain decode of a full batch at the benchmark's context
        dict(name="decode_b64_e4m3", kind="tree", B=64, N=1, Hq=32, Hkv=8, D=128, ctx=4096,
             ragged=True, e4m3=True, window=0, sinks=0, cap=0.0, dtype="bfloat16"),
        # the benchmark's verification step
        dict(name="tree_b16_e4m3", kind="tree", B=16, N=63, Hq=32, Hkv=8, D=128, ctx=4096,
             ragged=False, e4m3=True, window=0, sinks=0, cap=0.0, dtype="bfloat16"),
        # short prompts joining a step over 16-bit pages, the rest of one behind its first chunk
        dict(name="prompt_ragged_sinks", kind="prompt", lens="311 1 700 64 17", ctx="0 900 512 0 77",
             Hq=32, Hkv=8, D=64, e4m3=False, window=200, sinks=20, cap=0.0, dtype="float16", pad=3),
        # one long prompt
        dict(name="prompt_8k_e4m3", kind="prompt", lens="8192", ctx="0", Hq=32, Hkv=8, D=128,
             e4m3=True, window=0, sinks=0, cap=0.0, dtype="bfloat16", pad=0),
        # one user's next token at the small test models' vocabulary
        dict(name="logits_r1", kind="logits", B=1, N=0, V=32000, L=700, bias=0, masks=0,
             dtype="float32", to32=False),
        # a step's requests: biases, and a grammar for some of them
        dict(name="logits_r64_grammar", kind="logits", B=64, N=0, V=128256, L=2000, bias=100,
             masks=24, dtype="bfloat16", to32=False),
        # the benchmark's trees, every node behind its own path, as verification takes them
        dict(name="logits_tree_b8", kind="logits", B=8, N=63, V=128256, L=2000, bias=0, masks=0,
             dtype="bfloat16", to32=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(values):
    return " ".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split()]


def draw(rng):
    kind = rng.choice(["write", "read", "tree", "tree", "prompt", "logits"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    D = rng.choice([128, 128, 64])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (16, 16), (16, 8), (8, 1)])
    if kind in ("write", "read"):
        lens = [_log_int(rng, 1, 1600) for _ in range(rng.randint(1, 5))]
        if rng.random() < 0.4:
            lens = [rng.choice([1, 1, 7, 31, 63])] * _log_int(rng, 1, 64)
        pad = rng.choice([0, 0, 5])
        if kind == "read":
            return dict(kind=kind, lens=_text(lens), Hkv=Hkv, D=D, dtype=dtype, pad=pad,
                        starts=_text(rng.choice([0, _log_int(rng, 1, 2048)]) for _ in lens))
        return dict(kind=kind, lens=_text(lens), ctx=_log_int(rng, 1, 2048),
                    pos0=rng.choice([0, 0, 31000, 100000]), Hq=Hq, Hkv=Hkv, D=D,
                    layout=rng.choice(["half", "interleaved"]),
                    norm=rng.choice([True, True, False]), dtype=dtype, pad=pad)
    e4m3 = rng.choice([True, True, False])
    window = rng.choice([0, _log_int(rng, 1, 2048)]) if e4m3 else _log_int(rng, 1, 2048)
    sinks = rng.choice([1, 4, rng.randint(1, 200)]) if window else 0
    scores = dict(e4m3=e4m3, window=window, sinks=sinks, cap=rng.choice([0.0, 0.0, 50.0]),
                  dtype=dtype, Hq=Hq, Hkv=Hkv, D=D)
    if kind == "tree":
        N = rng.choice([1, 1, rng.randint(2, 63)])
        return dict(kind=kind, B=_log_int(rng, 1, 64 if N == 1 else 16), N=min(N, 256 * Hkv // Hq),
                    ctx=_log_int(rng, 64, 4096), ragged=rng.choice([True, False]), **scores)
    if kind == "prompt":
        n = rng.randint(1, 6)
        return dict(kind=kind, lens=_text(_log_int(rng, 1, 2600) for _ in range(n)),
                    ctx=_text(rng.choice([0, 0, _log_int(rng, 1, 2048)]) for _ in range(n)),
                    pad=rng.choice([0, 0, 5]), **scores)
    N = rng.choice([0, 0, rng.randint(1, 63)])
    B = _log_int(rng, 1, 64 if not N else 8)
    return dict(kind=kind, B=B, N=N, V=_log_int(rng, 8000, 128256), L=_log_int(rng, 1, 8000),
                bias=rng.choice([0, _log_int(rng, 1, 300)]), masks=rng.choice([0, rng.randint(1, B)]),
                dtype=rng.choice(["float32", "bfloat16", "float16"]),
                to32=rng.choice([False, True]))


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


# -- the pages ---------------------------------------------------------------------

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


def _quantise(x):
    """e4m3 codes of x [.., D] fp32 and the scales' bytes [..]: the smallest power
    of two 2^(byte - 127) that brings a row's largest magnitude to 448 or less."""
    top = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    m, e = torch.frexp(top)
    byte = torch.where(top > 0, e - torch.where(m <= TOP / 512, 9, 8) + 127, 1).clamp(min=1)
    codes = torch.ldexp(x, (127 - byte)[..., None]).to(torch.float8_e4m3fn)
    return codes, byte.to(torch.uint8)


def _values(codes, bytes_):
    """What codes [.., D] stand for, fp32."""
    return torch.ldexp(codes.float(), (bytes_.int() - 127)[..., None])


def _pools(case, nblk, g):
    """Pools and, of e4m3 ones, scales; keys and values of rows of different sizes."""
    shape = (nblk, 1, case["Hkv"], PAGE, case["D"])
    out = []
    for spread in (0.2, 1.0):
        size = torch.exp2(torch.randn(shape[:4], device="cuda", generator=g) * spread)
        x = torch.randn(shape, device="cuda", generator=g) * size[..., None]
        out.append(_quantise(x) if case.get("e4m3", True)
                   else (x.to(getattr(torch, case["dtype"])), None))
    (k, ks), (v, vs) = out
    return dict(kp=k, ks=ks, vp=v, vs=vs)


def _slots(s, seq, slot):
    """Blocks and offsets of slots [..] of sequences [..]."""
    return s["tables"][seq, slot // PAGE].long(), slot % PAGE


def _rows(s, which, block, off):
    """fp32 rows [.., Hkv, D] of the keys ("k") or values ("v") at blocks and offsets."""
    rows = s[which + "p"][block, 0, :, off]
    if s[which + "s"] is None:
        return rows.float()
    return _values(rows, s[which + "s"][block, 0, :, off])


def _packed(s):
    """Sequence and place in it of each packed token."""
    n = int(s["cu_host"][-1])
    lens = (s["cu"][1:] - s["cu"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(lens.numel(), device="cuda"), lens, output_size=n)
    return seq, torch.arange(n, device="cuda") - s["cu"].long()[seq]


def _cu(lens):
    return np.concatenate([[0], np.cumsum(lens)]).tolist()


# -- writing e4m3 pages, and reading them back --------------------------------------

def _prepare_write(case, g):
    lens, ctx, Hq, Hkv, D = _ints(case["lens"]), *(case[k] for k in ("ctx", "Hq", "Hkv", "D"))
    dt = getattr(torch, case["dtype"])
    B, T = len(lens), sum(lens) + case["pad"]
    base = [max(1, ctx - 5 * b) for b in range(B)]
    tables, nblk = _tables([c + n for c, n in zip(base, lens)], g)
    cu = _cu(lens)
    pos = np.zeros(T, np.int64)
    for b in range(B):
        pos[cu[b]: cu[b + 1]] = case["pos0"] + base[b] + np.arange(lens[b])
    norms = [(1.0 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dt) for _ in range(2)]
    s = dict(case=case, pos=_int32(pos.tolist()), cu=_int32(cu), cu_host=cu, base=_int32(base),
             tables=tables, norms=norms if case["norm"] else [None, None],
             qkv=torch.randn(T, (Hq + 2 * Hkv) * D, device="cuda", generator=g).to(dt),
             q_out=torch.zeros(T, Hq, D, dtype=dt, device="cuda"),
             k_out=torch.zeros(T, Hkv, D, dtype=dt, device="cuda"),
             v_out=torch.zeros(T, Hkv, D, dtype=dt, device="cuda"), **_pools(case, nblk, g))
    if own:
        from cudaforge_amd.rotary import Rotary

        s["rotary"] = Rotary(D, THETA, layout=case["layout"], device="cuda")
    return s


def _heads(s):
    case = s["case"]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    x = s["qkv"].view(-1, Hq + 2 * Hkv, D)
    return x[:, :Hq], x[:, Hq: Hq + Hkv], x[:, Hq + Hkv:]


def _run_write(s):
    case = s["case"]
    q, k, v = _heads(s)
    if own:
        from cudaforge_amd.rotary import qk_norm_rope_kv
        from cudaforge_amd.verify import kv_gather

        # sequences of one length need no table of where each begins
        cu = None if len(set(_ints(case["lens"]))) == 1 and not case["pad"] else s["cu"]
        qk_norm_rope_kv(q, k, v, s["pos"], s["rotary"], s["kp"], s["vp"], s["tables"], s["base"],
                        cu_seqlens=cu, q_norm=s["norms"][0], k_norm=s["norms"][1], eps=EPS,
                        q_out=s["q_out"], k_scales=s["ks"], v_scales=s["vs"])
        kv_gather(s["kp"], s["vp"], s["tables"], s["base"], cu_seqlens=cu, k_scales=s["ks"],
                  v_scales=s["vs"], k_out=s["k_out"], v_out=s["v_out"])
        return dict(q=s["q_out"], keys=s["k_out"], values=s["v_out"])
    n, D = s["cu_host"][-1], case["D"]
    i = torch.arange(0, D, 2, dtype=torch.float64, device="cuda")
    ang = s["pos"][:n].double()[:, None] * THETA ** (-i / D)
    cos, sin = ang.cos().float()[:, None, :], ang.sin().float()[:, None, :]

    def turned(x, w):
        x = x[:n].float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        if case["layout"] == "half":
            a, b = x[..., : D // 2], x[..., D // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)

    s["q_out"][:n] = turned(q, s["norms"][0]).to(s["q_out"].dtype)
    seq, place = _packed(s)
    block, off = _slots(s, seq, s["base"].long()[seq] + place)
    for which, x in (("k", turned(k, s["norms"][1])), ("v", v[:n].float())):
        codes, bytes_ = _quantise(x)
        s[which + "p"].view(torch.uint8)[block, 0, :, off] = codes.view(torch.uint8)
        s[which + "s"][block, 0, :, off] = bytes_
        s[which + "_out"][:n] = _rows(s, which, block, off).to(s[which + "_out"].dtype)
    return dict(q=s["q_out"], keys=s["k_out"], values=s["v_out"])


def _work_write(case):
    T, D = sum(_ints(case["lens"])), case["D"]
    Hq, Hkv = case["Hq"], case["Hkv"]
    # q in and out; k and v in, out as bytes with their scales, in again and out
    return {"bytes": T * (4 * Hq * D + 2 * Hkv * (2 * D + 2 * (D + 1) + 2 * D)),
            "flops": 10 * T * (Hq + Hkv) * D + 8 * T * Hkv * D}


def _grid64(x):
    """x [.., D] fp64 rounded to what e4m3 with the row's scale holds, by its
    definition: steps of 2^(e - 3) in the binade 2^e, of 2^-9 below 2^-6."""
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(top / TOP)).clamp(min=-126.0))
    # (log2 of a quotient next to a power of two may fall on either side)
    scale = torch.where(top > TOP * scale, scale * 2, scale)
    scale = torch.where((top <= TOP * scale / 2) & (scale > 2.0 ** -126), scale / 2, scale)
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def _exact_write(case, s):
    n, D = s["cu_host"][-1], case["D"]
    inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    ang = torch.outer(s["pos"][:n].double(), inv)
    # each pair as a complex number turned by its angle
    turn = torch.polar(torch.ones_like(ang), ang).unsqueeze(1)
    i = torch.arange(D // 2, device="cuda")
    a, b = (i, i + D // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
    out = []
    for x, w in zip(_heads(s)[:2], s["norms"]):
        y = x[:n].double()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        z = torch.complex(y[..., a], y[..., b]) * turn
        y = y.clone()
        y[..., a], y[..., b] = z.real, z.imag
        out.append(y)
    res = dict(q=s["q_out"].double(), keys=s["k_out"].double(), values=s["v_out"].double())
    res["q"][:n] = out[0]
    res["keys"][:n] = _grid64(out[1])
    res["values"][:n] = _grid64(_heads(s)[2][:n].double())
    return res


def _prepare_read(case, g):
    lens, starts, Hkv, D = _ints(case["lens"]), _ints(case["starts"]), case["Hkv"], case["D"]
    tables, nblk = _tables([c + n for c, n in zip(starts, lens)], g)
    T, cu = sum(lens) + case["pad"], _cu(lens)
    dt = getattr(torch, case["dtype"])
    return dict(case=case, cu=_int32(cu), cu_host=cu, base=_int32(starts), tables=tables,
                k_out=torch.zeros(T, Hkv, D, dtype=dt, device="cuda"),
                v_out=torch.zeros(T, Hkv, D, dtype=dt, device="cuda"), **_pools(case, nblk, g))


def _run_read(s):
    case = s["case"]
    if own:
        from cudaforge_amd.verify import kv_gather

        cu = None if len(set(_ints(case["lens"]))) == 1 and not case["pad"] else s["cu"]
        k, v = kv_gather(s["kp"], s["vp"], s["tables"], s["base"], cu_seqlens=cu,
                         k_scales=s["ks"], v_scales=s["vs"], k_out=s["k_out"], v_out=s["v_out"])
        return dict(keys=k, values=v)
    seq, place = _packed(s)
    block, off = _slots(s, seq, s["base"].long()[seq] + place)
    for which in "kv":
        out = s[which + "_out"]
        out[: seq.numel()] = _rows(s, which, block, off).to(out.dtype)
    return dict(keys=s["k_out"], values=s["v_out"])


def _work_read(case):
    T, D = sum(_ints(case["lens"])), case["D"]
    return {"bytes": 2 * T * case["Hkv"] * (D + 1 + 2 * D), "flops": 2 * T * case["Hkv"] * D}


def _values64(codes, bytes_):
    """What codes stand for, from their bits: sign, four of exponent, three of mantissa."""
    c = codes.view(torch.uint8).long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (1.0 + m / 8) * torch.exp2(e.double() - 7), m * 2.0 ** -9)
    return torch.where(c >= 128, -v, v) * torch.exp2(bytes_.double() - 127)[..., None]


def _pool64(s, which):
    pool = s[which + "p"][:, 0]
    return (pool.double() if s[which + "s"] is None
            else _values64(pool, s[which + "s"][:, 0]))


def _sequence64(pool, table, lo, hi):
    """Slots lo .. hi - 1 of a sequence, [Hkv, hi - lo, D]."""
    x = pool[table[: (hi + PAGE - 1) // PAGE].long()]
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, lo:hi]


def _exact_read(case, s):
    res = {}
    for which, name in (("k", "keys"), ("v", "values")):
        pool, out = _pool64(s, which), s[which + "_out"].double()
        for b, (n, c) in enumerate(zip(_ints(case["lens"]), _ints(case["starts"]))):
            at = s["cu_host"][b]
            out[at: at + n] = _sequence64(pool, s["tables"][b], c, c + n).transpose(0, 1)
        res[name] = out
    return res


# -- attention with a window and first tokens ---------------------------------------

def _ancestors(N):
    """[N] int: bit j of entry i says that node j is i or above it, in the
    complete binary tree numbered level by level."""
    masks = []
    for i in range(N):
        masks.append((masks[(i - 1) // 2] if i else 0) | (1 << i))
    return masks


def _mask_tensor(N):
    return torch.tensor(np.array(_ancestors(N), dtype=np.uint64).view(np.int64), device="cuda")


def _prepare_tree(case, g):
    B, N, Hq, D, ctx = (case[k] for k in ("B", "N", "Hq", "D", "ctx"))
    lens = torch.full((B,), ctx, dtype=torch.int32, device="cuda")
    if case["ragged"] and B > 1:
        lens = torch.randint(max(1, ctx // 4), ctx + 1, (B,), device="cuda", generator=g).int()
        lens[0] = ctx
    host = lens.tolist()
    tables, nblk = _tables([n + N for n in host], g)
    q = torch.randn(B, N, Hq, D, device="cuda", generator=g) * 2.0
    return dict(case=case, q=q.to(getattr(torch, case["dtype"])), tables=tables, lens=lens,
                host=host, masks=_mask_tensor(N), **_pools(case, nblk, g))


def _cache_args(s):
    case = s["case"]
    return dict(soft_cap=case["cap"], window=case["window"], sinks=case["sinks"],
                k_scales=s["ks"], v_scales=s["vs"])


def _seen(case, dist, slot, see):
    """What the window and the first tokens leave of the mask `see`."""
    if case["window"]:
        see = see & ((dist < case["window"]) | (slot < case["sinks"]))
    return see


def _attend(s, q, dist, see, longest):
    """q [B, n, Hq, D] over the first `longest` slots of each sequence, dist and see
    [B, n, longest]; fp32 [B, n, Hq, D]."""
    case = s["case"]
    B, n, Hq, D = q.shape
    Hkv = case["Hkv"]
    G = Hq // Hkv
    slot = torch.arange(longest, device="cuda")
    table = s["tables"][:, slot // PAGE].long().clamp(min=0)
    off = (slot % PAGE).expand(B, longest)
    see = _seen(case, dist, slot, see)[:, None, None]
    qh = q.float().view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    # (slots that a sequence does not have hold another's page: hidden by `see`)
    kh = _rows(s, "k", table, off).permute(0, 2, 3, 1).contiguous()
    sc = (qh @ kh).view(B, Hkv, G, n, longest) * (D ** -0.5)
    if case["cap"]:
        sc = torch.tanh(sc / case["cap"]) * case["cap"]
    sc = torch.where(see, sc, float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top > float("-inf"), top, 0.0))
    del sc
    total = p.sum(-1, keepdim=True)
    vh = _rows(s, "v", table, off).permute(0, 2, 1, 3).contiguous()
    o = (p.view(B, Hkv, G * n, longest) @ vh).view(B, Hkv, G, n, D)
    o = o / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)


def _run_tree(s):
    case = s["case"]
    N = case["N"]
    if own:
        from cudaforge_amd.verify import tree_attention

        return tree_attention(s["q"], s["kp"], s["vp"], s["tables"], s["lens"], s["masks"],
                              max_keys=case["ctx"] + N, **_cache_args(s))
    bits = (s["masks"][:, None] >> torch.arange(N, device="cuda")) & 1
    depth = bits.sum(-1) - 1
    longest = case["ctx"] + N
    ctx = s["lens"].long()[:, None]
    node = torch.arange(longest, device="cuda") - ctx                 # [B, S]
    inside = node.clamp(0, N - 1)
    at = torch.where(node < 0, node + ctx, ctx + depth[inside])       # positions of the keys
    see = (node < 0)[:, None] | ((node < N)[:, None]
                                 & bits[:, inside].bool().transpose(0, 1)
                                 & (node >= 0)[:, None])
    dist = (ctx + depth)[:, :, None] - at[:, None]
    return _attend(s, s["q"], dist, see, longest).to(s["q"].dtype)


def _attention_work(case, queries, pairs, keys):
    D = case["D"]
    row = D + 1 if case["e4m3"] else 2 * D
    return {"bytes": 2 * case["Hkv"] * keys * row + 4 * queries * case["Hq"] * D,
            "flops": 4 * case["Hq"] * D * pairs}


def _behind(ctx, W, sinks):
    """How many of the ctx slots in front a query sees whose window holds W of them."""
    return ctx if W >= ctx else W + min(sinks, ctx - W)


def _work_tree(case):
    B, N, W = case["B"], case["N"], case["window"] or 1 << 30
    depths = [bin(m).count("1") - 1 for m in _ancestors(N)]
    lens = [case["ctx"]] * B
    if case["ragged"] and B > 1:
        lens[1:] = [int(0.625 * case["ctx"])] * (B - 1)
    pairs = keys = 0
    for ctx in lens:
        behind = [_behind(ctx, max(0, W - 1 - d), case["sinks"]) for d in depths]
        pairs += sum(min(d + 1, W) for d in depths) + sum(behind)
        keys += max(behind) + N
    return _attention_work(case, B * N, pairs, keys)


def _attend64(case, q, k, v, dist, see):
    """q [n, Hq, D] over k, v [Hkv, S, D] fp64, some queries at a time, from the
    shares exp(score) / sum of them."""
    n, Hq, D = q.shape
    G = Hq // k.shape[0]
    out = torch.zeros(n, Hq, D, dtype=torch.float64, device="cuda")
    slot = torch.arange(k.shape[1], device="cuda")
    for lo in range(0, n, 512):
        rows = slice(lo, min(n, lo + 512))
        hidden = ~see[rows]
        if case["window"] > 0:
            hidden = hidden | ((dist[rows] >= case["window"]) & (slot >= case["sinks"]))
        for h in range(Hq):
            sc = torch.mm(q[rows, h].double(), k[h // G].t()) / math.sqrt(D)
            if case["cap"] > 0:
                e = torch.exp(-2.0 * sc.abs() / case["cap"])
                sc = case["cap"] * sc.sign() * (1.0 - e) / (1.0 + e)
            share = torch.softmax(sc.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
            out[rows, h] = torch.mm(share, v[h // G])
    return out


def _exact_tree(case, s):
    N, B = case["N"], case["B"]
    anc = _ancestors(N)
    tree = torch.tensor([[(m >> j) & 1 == 1 for j in range(N)] for m in anc], device="cuda")
    depth = torch.tensor([bin(m).count("1") - 1 for m in anc], device="cuda")
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    kp, vp = _pool64(s, "k"), _pool64(s, "v")
    for b in range(B):
        ctx = s["host"][b]
        see = torch.ones(N, ctx + N, dtype=torch.bool, device="cuda")
        see[:, ctx:] = tree
        far = torch.empty(N, ctx + N, dtype=torch.int64, device="cuda")
        far[:, :ctx] = ctx + depth[:, None] - torch.arange(ctx, device="cuda")
        far[:, ctx:] = depth[:, None] - depth
        out[b] = _attend64(case, s["q"][b], _sequence64(kp, s["tables"][b], 0, ctx + N),
                           _sequence64(vp, s["tables"][b], 0, ctx + N), far, see)
    return out


def _prepare_prompt(case, g):
    lens, ctx, Hq, D = _ints(case["lens"]), _ints(case["ctx"]), case["Hq"], case["D"]
    tables, nblk = _tables([c + n for c, n in zip(ctx, lens)], g)
    T, cu = sum(lens) + case["pad"], _cu(lens)
    q = torch.randn(T, Hq, D, device="cuda", generator=g) * 2.0
    q = q.to(getattr(torch, case["dtype"]))
    return dict(case=case, q=q, tables=tables, ctx=_int32(ctx), cu=_int32(cu), cu_host=cu,
                max_keys=max(c + n for c, n in zip(ctx, lens)), max_query=max(lens),
                out=torch.zeros_like(q), **_pools(case, nblk, g))


def _run_prompt(s):
    case = s["case"]
    if own:
        from cudaforge_amd.verify import prompt_attention

        return prompt_attention(s["q"], s["kp"], s["vp"], s["tables"], s["ctx"], s["cu"],
                                max_query=s["max_query"], max_keys=s["max_keys"], out=s["out"],
                                **_cache_args(s))
    # the chunks side by side, padded to the longest
    seq, place = _packed(s)
    B, n = len(_ints(case["lens"])), s["max_query"]
    q = torch.zeros(B, n, case["Hq"], case["D"], dtype=s["q"].dtype, device="cuda")
    q[seq, place] = s["q"][: seq.numel()]
    pos = s["ctx"].long()[:, None] + torch.arange(n, device="cuda")
    dist = pos[:, :, None] - torch.arange(s["max_keys"], device="cuda")
    out = _attend(s, q, dist, dist >= 0, s["max_keys"])
    s["out"][: seq.numel()] = out[seq, place].to(s["out"].dtype)
    return s["out"]


def _work_prompt(case):
    pairs = keys = 0
    W = case["window"] or 1 << 30
    for n, ctx in zip(_ints(case["lens"]), _ints(case["ctx"])):
        pairs += sum(_behind(ctx + i + 1, W, case["sinks"]) for i in range(n))
        keys += min(ctx + n, n + W - 1 + case["sinks"])
    return _attention_work(case, sum(_ints(case["lens"])), pairs, keys)


def _exact_prompt(case, s):
    out = s["out"].double()
    kp, vp = _pool64(s, "k"), _pool64(s, "v")
    for b, (n, ctx) in enumerate(zip(_ints(case["lens"]), _ints(case["ctx"]))):
        t0 = s["cu_host"][b]
        key = torch.arange(ctx + n, device="cuda")
        far = ctx + key[:n].unsqueeze(1) - key
        out[t0: t0 + n] = _attend64(case, s["q"][t0: t0 + n],
                                    _sequence64(kp, s["tables"][b], 0, ctx + n),
                                    _sequence64(vp, s["tables"][b], 0, ctx + n), far, far >= 0)
    return out


# -- logits in front of the sampler ---------------------------------------------------

def _prepare_logits(case, g):
    B, N, V, L = (case[k] for k in ("B", "N", "V", "L"))
    R = (B, N, V) if N else (B, V)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, device="cuda", generator=g, dtype=torch.int32)

    # conversations repeat themselves: half their tokens come from a few
    common = ints(0, V, 64)
    history = torch.where(torch.rand(B, L, device="cuda", generator=g) < 0.5, ints(0, V, B, L),
                          common[ints(0, 64, B, L).long()])
    lens = ints(max(1, L // 3), L + 1, B)
    lens[0] = L
    prompt = (lens * torch.rand(B, device="cuda", generator=g)).int()

    def pick(values):
        at = torch.randint(0, len(values), (B,), device="cuda", generator=g)
        return torch.tensor(values, dtype=torch.float32, device="cuda")[at]

    s = dict(case=case, logits=(torch.randn(R, device="cuda", generator=g) * 3.0).to(
                 getattr(torch, case["dtype"])),
             history=history, history_lens=lens, prompt_lens=prompt,
             repetition=pick([1.0, 1.1, 1.3]), frequency=pick([0.0, 0.2, 0.7]),
             presence=pick([0.0, 0.4]), nodes=None, masks=None, bias_tokens=None,
             bias_values=None, allowed=None, allowed_index=None)
    if N:
        s["nodes"] = torch.where(torch.rand(B, N, device="cuda", generator=g) < 0.5,
                                 ints(0, V, B, N), common[ints(0, 64, B, N).long()])
        s["masks"] = _mask_tensor(N)
    if case["bias"]:
        # distinct tokens, -1 behind each request's own
        K = case["bias"]
        pool = torch.randperm(V, device="cuda", generator=g)[:K].int()
        used = torch.arange(K, device="cuda") < ints(0, K + 1, B, 1)
        s["bias_tokens"] = torch.where(used, pool, -1)
        s["bias_values"] = torch.randn(B, K, device="cuda", generator=g) * 2.0
    if case["masks"]:
        # grammars' masks, and which one each row stands in (-1: none)
        M = case["masks"]
        s["allowed"] = ints(-2 ** 31, 2 ** 31 - 1, M, (V + 31) // 32)
        s["allowed_index"] = ints(-1, M, *R[:-1])
    return s


def _run_logits(s):
    case = s["case"]
    B, N, V = case["B"], case["N"], case["V"]
    if own:
        from cudaforge_amd.sampling import adjust_logits

        return adjust_logits(
            s["logits"], history=s["history"], history_lens=s["history_lens"],
            prompt_lens=s["prompt_lens"], repetition=s["repetition"], frequency=s["frequency"],
            presence=s["presence"], node_tokens=s["nodes"], tree_mask=s["masks"],
            bias_tokens=s["bias_tokens"], bias_values=s["bias_values"], allowed=s["allowed"],
            allowed_index=s["allowed_index"], out_dtype=torch.float32 if case["to32"] else None)
    rows = (-1,) + (1,) * (s["logits"].dim() - 1)
    at = torch.arange(case["L"], device="cuda")
    inside = at < s["history_lens"][:, None]
    made = inside & (at >= s["prompt_lens"][:, None])
    tokens = s["history"].long()
    count = torch.zeros(B, V, device="cuda").scatter_add_(1, tokens, made.float())
    seen = torch.zeros(B, V, device="cuda").scatter_add_(1, tokens, inside.float())
    if N:
        bits = ((s["masks"][:, None] >> torch.arange(N, device="cuda")) & 1).float()
        path = torch.zeros(B, N, V, device="cuda").scatter_add_(
            2, s["nodes"].long()[:, None, :].expand(B, N, N), bits.expand(B, N, N))
        count, seen = count[:, None] + path, seen[:, None] + path
    x = s["logits"].float()
    r = s["repetition"].view(rows)
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"].view(rows) * count - s["presence"].view(rows) * (count > 0)
    if case["bias"]:
        there = s["bias_tokens"] >= 0
        b = torch.zeros(B, V, device="cuda").scatter_add_(
            1, s["bias_tokens"].clamp(min=0).long(), torch.where(there, s["bias_values"], 0.0))
        x = x + (b[:, None] if N else b)
    if case["masks"]:
        v = torch.arange(V, device="cuda")
        index = s["allowed_index"].long()
        word = s["allowed"][index.clamp(min=0)][..., v // 32]
        ok = ((word >> (v % 32).int()) & 1).bool() | (index < 0)[..., None]
        x = torch.where(ok, x, float("-inf"))
    return x if case["to32"] else x.to(s["logits"].dtype)


def _work_logits(case):
    R, V = case["B"] * max(case["N"], 1), case["V"]
    size = 4 if case["dtype"] == "float32" else 2
    row = (size + (4 if case["to32"] else size)) * V
    if case["masks"]:
        row += V // 8
    return {"bytes": R * row + case["B"] * (4 * case["L"] + 8 * case["bias"]), "flops": 4 * R * V}


def _exact_logits(case, s):
    """Request by request, from each touched token's own counts."""
    B, N, V = case["B"], case["N"], case["V"]
    out = s["logits"].double().view(B, -1, V).clone()
    nodes = s["nodes"].tolist() if N else None
    anc = _ancestors(N) if N else [0]
    hist, lens, prompts = (s[k].tolist() for k in ("history", "history_lens", "prompt_lens"))
    for b in range(B):
        theta, freq, pres = (float(s[k][b]) for k in ("repetition", "frequency", "presence"))
        made, old = {}, set(hist[b][: lens[b]])
        for t in hist[b][prompts[b]: lens[b]]:
            made[t] = made.get(t, 0) + 1
        for i in range(max(N, 1)):
            counts = dict(made)
            for j in range(N):
                if (anc[i] >> j) & 1:
                    counts[nodes[b][j]] = counts.get(nodes[b][j], 0) + 1
            at = sorted(old | set(counts))
            where = torch.tensor(at, device="cuda")
            c = torch.tensor([counts.get(t, 0) for t in at], dtype=torch.float64, device="cuda")
            x = out[b, i, where]
            x = torch.where(x > 0, x / theta, x * theta) - freq * c - pres * (c > 0).double()
            out[b, i, where] = x
        if case["bias"]:
            for t, v in zip(s["bias_tokens"][b].tolist(), s["bias_values"][b].tolist()):
                if t >= 0:
                    out[b, :, t] += v
    out = out.view(s["logits"].shape)
    if case["masks"]:
        words = s["allowed"].cpu().numpy().view(np.uint8)
        bits = np.unpackbits(words, axis=1, bitorder="little")[:, :V] == 0
        hidden = torch.from_numpy(np.concatenate([bits, np.zeros((1, V), bool)])).cuda()
        out[hidden[s["allowed_index"].long()]] = -math.inf   # (-1: the last row, nothing)
    return out


_PREPARE = {"write": _prepare_write, "read": _prepare_read, "tree": _prepare_tree,
            "prompt": _prepare_prompt, "logits": _prepare_logits}
_RUN = {"write": _run_write, "read": _run_read, "tree": _run_tree, "prompt": _run_prompt,
        "logits": _run_logits}
_WORK = {"write": _work_write, "read": _work_read, "tree": _work_tree, "prompt": _work_prompt,
         "logits": _work_logits}
_EXACT = {"write": _exact_write, "read": _exact_read, "tree": _exact_tree,
          "prompt": _exact_prompt, "logits": _exact_logits}
