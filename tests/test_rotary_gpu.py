"""GPU tier: cfa_qk_norm_rope_kv against the formulas in 64 bits.

Tolerance: the one rounding to the 16-bit type, half a step (eps / 2 of the
value), plus the fp32 arithmetic's error, which is relative to the pair: about
four roundings of the norm (2^-24 each), the angle's conversion to fp32 turns
(2^-25 turn = 2^-22.3 radian), two units in the last place of sine and cosine
and three roundings of the turn; in all below 2^-20 (|a| + |b|)."""
import pytest
import torch

from cudaforge_amd.rotary import Rotary, qk_norm_rope_kv

pytestmark = pytest.mark.gpu


def _want(x, w, eps, pos, rotary, dtype):
    """fp64 result of x [T, H, D] and the bound of its error."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    mag = y.abs()
    if rotary is not None and rotary.rotary_dim:
        rot = rotary.rotary_dim
        ang = pos.double()[:, None] * rotary.radians
        cos, sin = (ang.cos() * rotary.factor)[:, None], (ang.sin() * rotary.factor)[:, None]
        i = torch.arange(rot // 2)
        ia, ib = (i, i + rot // 2) if rotary.layout == "half" else (2 * i, 2 * i + 1)
        a, b = y[..., ia], y[..., ib]
        y, mag = y.clone(), mag.clone()
        y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
        m = (a.abs() + b.abs()) * rotary.factor
        mag[..., ia], mag[..., ib] = m, m
    return y, torch.finfo(dtype).eps / 2 * y.abs() + 2.0 ** -20 * mag


def _case(dtype, lens, Hq, Hkv, D, bs=16, seed=0, layers=2, base=None, pad=0):
    g = torch.Generator().manual_seed(seed)
    B, T = len(lens), sum(lens) + pad
    base = base or [7 * b + 3 for b in range(B)]
    need = [(c + n + bs - 1) // bs for c, n in zip(base, lens)]
    perm = torch.randperm(sum(need) + 3, generator=g).int()
    bt = torch.full((B, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[at: at + n]
        at += n
    pools = [torch.randn(len(perm), layers, Hkv, bs, D, generator=g).to(dtype) for _ in range(2)]
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g).to(dtype)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)
    pos = torch.randint(0, 200000, (T,), generator=g, dtype=torch.int32)
    return qkv, pos, cu, torch.tensor(base, dtype=torch.int32), bt, pools


def _check(device, dtype, lens, Hq, Hkv, D, rotary, *, norm=None, eps=1e-6, ragged=True, layer=1,
           bs=16, pad=0, view=lambda x: x, pos=None, base=None, unmap=()):
    qkv, p, cu, base, bt, pools = _case(dtype, lens, Hq, Hkv, D, bs=bs, pad=pad, base=base)
    p = p if pos is None else pos
    for b, page in unmap:
        bt[b, page] = -1
    g = torch.Generator().manual_seed(9)
    wq = wk = None
    if norm is not None:
        wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(norm) for _ in range(2))
    d = view(qkv.to(device))
    kp, vp = (x.to(device) for x in pools)
    T = d.shape[0]
    q_out = torch.full((T, Hq, D), 5.0, dtype=dtype, device=device)
    got = qk_norm_rope_kv(
        d[:, :Hq], d[:, Hq: Hq + Hkv], d[:, Hq + Hkv:], p.to(device),
        None if rotary is None else rotary.to(device), kp, vp, bt.to(device), base.to(device),
        layer=layer, cu_seqlens=cu.to(device) if ragged else None,
        q_norm=None if wq is None else wq.to(device), k_norm=None if wk is None else wk.to(device),
        eps=eps, q_out=q_out)
    assert got is q_out
    n = int(cu[-1])
    q, tq = _want(qkv[:n, :Hq], wq, eps, p[:n], rotary, dtype)
    k, tk = _want(qkv[:n, Hq: Hq + Hkv], wk, eps, p[:n], rotary, dtype)
    out = got.cpu()
    assert ((out[:n].double() - q).abs() <= tq).all()
    assert (out[n:] == 5.0).all()                       # rows of no sequence
    kw, vw = (x.clone() for x in pools)
    kt = torch.zeros(kw.shape, dtype=torch.float64)
    kd = kw.double()
    for b, m in enumerate(lens):
        for j in range(m):
            slot = int(base[b]) + j
            blk = int(bt[b, slot // bs])
            if blk < 0:
                continue
            t = int(cu[b]) + j
            kd[blk, layer, :, slot % bs] = k[t]
            kt[blk, layer, :, slot % bs] = tk[t]
            vw[blk, layer, :, slot % bs] = qkv[t, Hq + Hkv:]
    assert ((kp.cpu().double() - kd).abs() <= kt).all()  # every other slot as it was
    assert torch.equal(vp.cpu().view(torch.int16), vw.view(torch.int16))


BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("D,rot", [(128, 128), (64, 64), (128, 64), (128, 32), (64, 16), (96, 96),
                                   (80, 80), (80, 40), (128, 100), (8, 8), (8, 2), (256, 256),
                                   (136, 136), (32, 32), (128, 0)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_head_sizes_and_parts(device, D, rot, layout):
    _check(device, BF, [5, 1, 18], 4, 2, D, Rotary(rot, 10000.0, layout=layout), norm=BF)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("norm", [None, "own", torch.float32])
@pytest.mark.parametrize("ragged", [True, False])
def test_types_and_norms(device, dtype, norm, ragged):
    _check(device, dtype, [3, 3, 3], 8, 2, 128, Rotary(128, 500000.0),
           norm=dtype if norm == "own" else norm, ragged=ragged)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (7, 1), (32, 8), (71, 1)])
def test_head_counts(device, Hq, Hkv):
    _check(device, BF, [2, 5], Hq, Hkv, 64, Rotary(64), norm=BF)


@pytest.mark.parametrize("lens,pad", [([1], 0), ([1] * 70, 0), ([0, 4, 0, 0, 9, 0], 5),
                                      ([700, 1, 400], 3), ([0], 2)])
def test_ragged_batches(device, lens, pad):
    """More than 64 sequences, empty ones, padding behind the last, and enough
    tokens for the variant of four rows a lane group."""
    _check(device, BF, lens, 8, 2, 128, Rotary(128, scaling=dict(kind="linear", factor=4.0)),
           norm=BF, pad=pad, layer=0)


@pytest.mark.parametrize("bs", [1, 5, 16, 32])
def test_page_sizes(device, bs):
    _check(device, BF, [9, 40], 4, 4, 64, Rotary(64), bs=bs)


def test_far_and_negative_positions(device):
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 131071, 1000003, 77], dtype=torch.int32)
    for layout in ("half", "interleaved"):
        _check(device, HF, [8], 4, 2, 128, Rotary(128, 500000.0, layout=layout), pos=pos)


def test_scaled_rotation(device):
    for sc in (dict(kind="yarn", factor=16.0, original=4096), dict(kind="ntk", factor=8.0),
               dict(kind="bands", factor=8.0, low=1.0, high=4.0, original=8192)):
        _check(device, BF, [30], 4, 2, 128, Rotary(128, 500000.0, scaling=sc), norm=BF)


def test_strided_and_unaligned_views(device):
    def wide(x):                       # a slice of a wider projection
        w = torch.zeros(x.shape[0], x.shape[1] + 3, x.shape[2], dtype=x.dtype, device=x.device)
        w[:, 1: 1 + x.shape[1]] = x
        return w[:, 1: 1 + x.shape[1]]

    def odd(x):                        # rows that begin at odd elements
        w = torch.zeros(x.shape[0], x.shape[1] * x.shape[2] + 1, dtype=x.dtype, device=x.device)
        w[:, 1:] = x.flatten(1)
        return w.as_strided(x.shape, (w.stride(0), x.shape[2], 1), 1)

    def heads_first(x):
        return x.transpose(0, 1).contiguous().transpose(0, 1)

    for view in (wide, odd, heads_first):
        for layout in ("half", "interleaved"):
            _check(device, BF, [5, 6], 4, 2, 64, Rotary(64, layout=layout), norm=BF, view=view)


def test_unmapped_pages_and_slots_outside_the_table(device):
    # page 1 of sequence 0 is not mapped; sequence 1 begins in front of slot 0
    _check(device, BF, [40, 5], 4, 2, 64, Rotary(64), unmap=[(0, 1)])
    qkv, p, cu, base, bt, pools = _case(BF, [40, 5], 4, 2, 64)
    d = qkv.to(device)
    kp, vp = (x.to(device) for x in pools)
    bt[0, 0] = 1000000                                  # outside the pool
    for start in ([-50, -50], [10 ** 6, 2 ** 31 - 3]):
        qk_norm_rope_kv(d[:, :4], d[:, 4:6], d[:, 6:], p.to(device), None, kp, vp,
                        bt[:, :1].contiguous().to(device),
                        torch.tensor(start, dtype=torch.int32, device=device),
                        cu_seqlens=cu.to(device))
    assert torch.equal(kp.cpu(), pools[0]) and torch.equal(vp.cpu(), pools[1])


def test_infinities_stay_in_their_pairs(device):
    """Elements behind the rotated ones are copied, infinite or not; v too."""
    qkv, p, cu, base, bt, pools = _case(BF, [2], 2, 1, 64)
    qkv[:, :, 63] = float("inf")
    qkv[:, 3, 0] = float("nan")
    d = qkv.to(device)
    kp, vp = (x.to(device) for x in pools)
    q = qk_norm_rope_kv(d[:, :2], d[:, 2:3], d[:, 3:], p.to(device), Rotary(32, device=device), kp,
                        vp, bt.to(device), base.to(device)).cpu()
    assert torch.isinf(q[..., 63]).all() and torch.isfinite(q[..., :63]).all()
    assert torch.isnan(vp.cpu()[int(bt[0, 0]), 0, 0, 3, 0])


def test_other_stream_and_graph(device):
    """On a stream of the caller's, and replayed with other inputs and lengths."""
    qkv, p, cu, base, bt, pools = _case(BF, [4, 4], 4, 2, 128)
    rot = Rotary(128, device=device)
    d, pd, bd, btd = (x.to(device) for x in (qkv, p, base, bt))

    def call(kp, vp, out):
        return qk_norm_rope_kv(d[:, :4], d[:, 4:6], d[:, 6:], pd, rot, kp, vp, btd, bd, q_out=out)

    side = torch.cuda.Stream(device)
    kp, vp = (x.to(device) for x in pools)
    out = torch.empty(8, 4, 128, dtype=BF, device=device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        call(kp, vp, out)
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(kp, vp, out)
    for step in range(3):
        d.copy_(torch.randn(d.shape, generator=torch.Generator().manual_seed(step)).to(BF))
        pd.add_(4)
        graph.replay()
        torch.cuda.synchronize()
        k2, v2 = (x.to(device) for x in pools)
        o2 = call(k2, v2, torch.empty_like(out))
        assert torch.equal(out, o2) and torch.equal(kp, k2) and torch.equal(vp, v2)
    graph.reset()


def test_refusals_on_the_device(device):
    qkv, p, cu, base, bt, pools = _case(BF, [4, 4], 4, 2, 64)
    d, pd, bd, btd = (x.to(device) for x in (qkv, p, base, bt))
    kp, vp = (x.to(device) for x in pools)
    rot = Rotary(64, device=device)
    ok = dict(q=d[:, :4], k=d[:, 4:6], v=d[:, 6:], positions=pd, rotary=rot, k_pool=kp, v_pool=vp,
              block_tables=btd, base_lens=bd)
    qk_norm_rope_kv(**ok)
    for bad in (dict(k=d[:, 4:5]), dict(v=d[:, 6:7]), dict(k=d[:, 4:6].half()),
                dict(positions=pd.long()), dict(positions=pd[:7]), dict(rotary=Rotary(64)),
                dict(rotary=Rotary(66, device=device)), dict(k_pool=kp.half()),
                dict(v_pool=vp[:1]), dict(k_pool=kp[..., :32]), dict(block_tables=btd[:1]),
                dict(base_lens=bd[:1]), dict(cu_seqlens=cu[:2].to(device)),
                dict(q=d[:, :4].transpose(1, 2)), dict(q_norm=torch.ones(32, device=device)),
                dict(q_norm=torch.ones(64, device=device), k_norm=torch.ones(64, device=device, dtype=BF)),
                dict(q_out=torch.empty(8, 4, 64, device=device)), dict(layer=2), dict(eps=-1.0),
                dict(q_out=d.flatten()[: 8 * 4 * 64].view(8, 4, 64))):
        with pytest.raises(ValueError):
            qk_norm_rope_kv(**{**ok, **bad})
    empty = qk_norm_rope_kv(**{**ok, "q": d[:0, :4], "k": d[:0, 4:6], "v": d[:0, 6:],
                               "positions": pd[:0]})
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("D,rot,layout,norm", [
    (128, 128, "half", True), (128, 128, "interleaved", False), (128, 100, "half", True),
    (64, 32, "half", False), (256, 256, "half", True)])
@pytest.mark.parametrize("T", [700, 2800, 9001])
def test_large_batches_are_small_ones(device, D, rot, layout, norm, T):
    """A row is the same bits whatever its batch (which sets how many rows a wave
    takes): one call against calls of 100 tokens."""
    Hq, Hkv, bs = 16, 2, 16
    g = torch.Generator(device=device).manual_seed(21)
    qkv = torch.randn(T, Hq + 2 * Hkv, D, device=device, generator=g).to(BF)
    w = (1 + 0.1 * torch.randn(D, device=device, generator=g)).to(BF) if norm else None
    pos = torch.randint(0, 100000, (T,), device=device, generator=g, dtype=torch.int32)
    rotary = Rotary(rot, layout=layout, device=device)
    pages = (T + bs - 1) // bs
    pools = [torch.full((pages, 1, Hkv, bs, D), 3.0, dtype=BF, device=device) for _ in range(4)]
    bt = torch.randperm(pages, device=device, generator=g).int().view(1, pages)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    zero = torch.zeros(1, dtype=torch.int32, device=device)
    got = qk_norm_rope_kv(q, k, v, pos, rotary, *pools[:2], bt, zero, q_norm=w, k_norm=w)
    want = torch.cat([
        qk_norm_rope_kv(q[t: t + 100], k[t: t + 100], v[t: t + 100], pos[t: t + 100], rotary,
                        *pools[2:], bt, zero + t, q_norm=w, k_norm=w) for t in range(0, T, 100)])
    assert torch.equal(got, want)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_offsets_past_32_bits(device):
    """Pages behind 2^31 elements of the pools, and q's tokens so far apart."""
    Hq, Hkv, D, bs, blocks = 4, 8, 128, 16, 140000
    g = torch.Generator(device=device).manual_seed(22)
    big = [torch.empty(blocks, 1, Hkv, bs, D, dtype=BF, device=device) for _ in range(2)]
    small = [torch.empty(3, 1, Hkv, bs, D, dtype=BF, device=device) for _ in range(2)]
    far = torch.empty((1 << 31) + 4096, dtype=BF, device=device)
    q = far.as_strided((3, Hq, D), ((1 << 30) + 128, D, 1))
    q.copy_(torch.randn(3, Hq, D, device=device, generator=g))
    k, v = (torch.randn(3, Hkv, D, device=device, generator=g).to(BF) for _ in range(2))
    pos = torch.tensor([5, 6, 70000], dtype=torch.int32, device=device)
    rotary = Rotary(D, device=device)
    base = torch.tensor([15], dtype=torch.int32, device=device)
    pages = [139998, 131073, 7]
    out = []
    for pools, table in ((big, pages), (small, [0, 1, 2])):
        bt = torch.tensor([table], dtype=torch.int32, device=device)
        out.append(qk_norm_rope_kv(q, k, v, pos, rotary, *pools, bt, base))
    assert torch.equal(*out)
    for b, s in zip(big, small):
        assert torch.equal(b[139998, :, :, 15], s[0, :, :, 15])
        assert torch.equal(b[131073, :, :, :2], s[1, :, :, :2])
    want = qk_norm_rope_kv(q.contiguous(), k, v, pos, rotary, *small,
                           torch.tensor([[0, 1, 2]], dtype=torch.int32, device=device), base)
    assert torch.equal(out[0], want)
