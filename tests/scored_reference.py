"""Plain 64-bit attention over paged caches with capped, biased and windowed
scores, and the error that the kernels' roundings may cause."""
import torch


def gather(pool, table, n, layer):
    """The first n slots of one sequence, fp64 [Hkv, n, D]."""
    bs = pool.shape[3]
    x = pool[table[: (n + bs - 1) // bs].long().clamp_min(0), layer]
    return x.transpose(0, 1).reshape(pool.shape[2], -1, pool.shape[4])[:, :n].double()


def attend(q, k, v, qpos, kpos, see, scale, cap=0.0, slopes=None, window=0, dtype=torch.bfloat16):
    """q [n, Hq, D], k / v [Hkv, S, D], positions [n] / [S], see [n, S] bool;
    returns the output [n, Hq, D] and its tolerance.

    A probability is rounded to 16 bits (u = eps / 2 of its value; in fp16 not
    finer than 2^-25 of the base, which no maximum falls short of), the row's
    sum is taken of the rounded ones, and the output is rounded once: u |out| +
    2 u A with A = sum p |v| / sum p.  A score is off by ds: D + 8 fp32
    roundings (2^-24) of its products, 2^-20 (polynomial, tanh and exp2) of
    itself, 2^-22 of the bias, and 2^-20 absolute; p by the factor e^ds, twice
    (values and sum).
    """
    n, Hq, D = q.shape
    G = Hq // k.shape[0]
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    tol = torch.zeros(n, Hq, D, dtype=torch.float64)
    if k.shape[1] == 0:
        return out, tol
    u = torch.finfo(dtype).eps / 2
    dist = (qpos[:, None] - kpos[None, :]).double()
    see = see & (dist < window) if window else see
    tiny = k.shape[1] * 2.0 ** -25 if dtype == torch.float16 else 0.0
    for h in range(Hq):
        kk, vv = k[h // G], v[h // G]
        s = q[:, h].double() @ kk.t() * scale
        mag = q[:, h].double().abs() @ kk.abs().t() * abs(scale)
        if cap:
            s = cap * torch.tanh(s / cap)
        bias = torch.zeros_like(s) if slopes is None else -float(slopes[h]) * dist
        s = (s + bias).masked_fill(~see, float("-inf"))
        some = see.any(-1)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        o = p @ vv.masked_fill(~see.any(0)[:, None], 0.0)
        o[~some] = 0.0
        ds = (D + 8) * 2.0 ** -24 * mag + 2.0 ** -20 * (s.abs().nan_to_num(0.0, 0.0, 0.0) + 1.0) \
            + 2.0 ** -22 * bias.abs()
        ds = (ds * (p > 1e-9)).max(-1, keepdim=True).values
        A = p @ vv.abs().nan_to_num(0.0, 0.0, 0.0)
        out[:, h] = o
        tol[:, h] = u * o.abs() + 2 * (u + ds) * A + 2 * tiny * vv.abs().nan_to_num(0., 0., 0.).max() \
            + 1e-30
        tol[:, h] += u * tol[:, h]
    return out, tol


def tree_case(lens, N, Hq, Hkv, D, dtype, *, bs=16, layers=1, seed=0, qscale=2.0):
    """q [B, N, Hq, D], pools, block tables (-1 behind a sequence's pages)."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + N + bs - 1) // bs for n in lens]
    nblk = sum(need) + 2
    perm = torch.randperm(nblk, generator=g).int()
    bt = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[at: at + n]
        at += n
    kp, vp = (torch.randn(nblk, layers, Hkv, bs, D, generator=g).to(dtype) for _ in range(2))
    q = (qscale * torch.randn(len(lens), N, Hq, D, generator=g)).to(dtype)
    return q, kp, vp, bt


def tree_want(q, kp, vp, bt, lens, masks, *, layer=0, scale=None, first=0, **score):
    """masks: python ints of all N nodes (one list, or one a sequence)."""
    B, Nq, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    outs, tols = [], []
    for b, ctx in enumerate(lens):
        m = masks[b] if isinstance(masks[0], (list, tuple)) else masks
        N = len(m)
        see = torch.tensor([[(m[i] >> j) & 1 == 1 for j in range(N)] for i in range(first, N)])
        depth = torch.tensor([max(bin(x).count("1") - 1, 0) for x in m])
        see = torch.cat([torch.ones(Nq, ctx, dtype=torch.bool), see], 1)
        kpos = torch.cat([torch.arange(ctx), ctx + depth])
        o, t = attend(q[b], gather(kp, bt[b], ctx + N, layer), gather(vp, bt[b], ctx + N, layer),
                      ctx + depth[first:], kpos, see, scale, dtype=q.dtype, **score)
        outs.append(o)
        tols.append(t)
    return torch.stack(outs), torch.stack(tols)


def prompt_want(q, kp, vp, bt, ctx, lens, *, layer=0, scale=None, **score):
    Hq, D = q.shape[1:]
    scale = D ** -0.5 if scale is None else scale
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    t0 = 0
    for b, (c, n) in enumerate(zip(ctx, lens)):
        kpos = torch.arange(c + n)
        qpos = torch.arange(c, c + n)
        out[t0: t0 + n], tol[t0: t0 + n] = attend(
            q[t0: t0 + n], gather(kp, bt[b], c + n, layer), gather(vp, bt[b], c + n, layer), qpos,
            kpos, qpos[:, None] >= kpos, scale, dtype=q.dtype, **score)
        t0 += n
    return out, tol
