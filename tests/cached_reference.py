"""Plain 64-bit attention over paged caches of 16 bits or of e4m3 codes, through a
window with first tokens that stay visible; errors as in scored_reference.attend."""
import torch

from tests import e4m3_reference as E
from tests import scored_reference as R


def case(lens, extra, Hkv, D, dtype, *, e4m3, bs=16, layers=1, seed=0):
    """Pools ((codes, scales), or (16-bit, None)) of K and V and block tables for
    sequences of lens[b] + extra slots (a number, or one each)."""
    g = torch.Generator().manual_seed(seed)
    extra = [extra] * len(lens) if isinstance(extra, int) else extra
    need = [(n + x + bs - 1) // bs for n, x in zip(lens, extra)]
    nblk = sum(need) + 2
    perm = torch.randperm(nblk, generator=g).int()
    bt = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[at: at + n]
        at += n
    shape = (nblk, layers, Hkv, bs, D)
    if e4m3:
        pools = [E.random_pool(shape, g, spread) for spread in (0.2, 2.0)]
    else:
        pools = [(torch.randn(shape, generator=g).to(dtype), None) for _ in range(2)]
    return pools, bt


def rows(pool, table, n, layer):
    codes, scales = pool
    x = codes if scales is None else E.values(codes[:, layer], scales[:, layer])[:, None]
    return R.gather(x, table, n, layer if scales is None else 0)


def attend(q, k, v, qpos, kpos, see, scale, *, window=0, sinks=0, dtype, **score):
    if window:
        near = qpos[:, None] - kpos[None, :] < window
        see = see & (near | (torch.arange(kpos.numel()) < sinks))
    return R.attend(q, k, v, qpos, kpos, see, scale, dtype=dtype, **score)


def tree_want(q, pools, bt, lens, masks, *, layer=0, first=0, **kw):
    B, Nq, Hq, D = q.shape
    outs, tols = [], []
    N = len(masks)
    for b, ctx in enumerate(lens):
        see = torch.tensor([[(masks[i] >> j) & 1 == 1 for j in range(N)] for i in range(first, N)])
        depth = torch.tensor([max(bin(x).count("1") - 1, 0) for x in masks])
        see = torch.cat([torch.ones(Nq, ctx, dtype=torch.bool), see], 1)
        kpos = torch.cat([torch.arange(ctx), ctx + depth])
        k, v = (rows(p, bt[b], ctx + N, layer) for p in pools)
        o, t = attend(q[b], k, v, ctx + depth[first:], kpos, see, D ** -0.5, dtype=q.dtype, **kw)
        outs.append(o)
        tols.append(t)
    return torch.stack(outs), torch.stack(tols)


def prompt_want(q, pools, bt, ctx, lens, *, layer=0, **kw):
    Hq, D = q.shape[1:]
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    t0 = 0
    for b, (c, n) in enumerate(zip(ctx, lens)):
        kpos, qpos = torch.arange(c + n), torch.arange(c, c + n)
        k, v = (rows(p, bt[b], c + n, layer) for p in pools)
        out[t0: t0 + n], tol[t0: t0 + n] = attend(q[t0: t0 + n], k, v, qpos, kpos,
                                                  qpos[:, None] >= kpos, D ** -0.5, dtype=q.dtype,
                                                  **kw)
        t0 += n
    return out, tol
