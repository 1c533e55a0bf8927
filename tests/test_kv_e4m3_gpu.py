"""GPU tier: the 8-bit paged cache: rows quantised as they are written, read
back, and moved with their scales.

v is quantised from the 16-bit values: every bit is fixed.  k comes out of the
norm and the rotation in fp32, off by 2^-20 (|a| + |b|) of the formula in 64 bits
(the bound that tests/test_rotary_gpu.py derives): its code is that of some value
so near, half a step of the code off at most; its scale that of a largest value so
near."""
import pytest
import torch

from cudaforge_amd.kv_cache import KVCacheConfig, PagedKVCache
from cudaforge_amd.rotary import Rotary, qk_norm_rope_kv
from cudaforge_amd.verify import kv_commit, kv_gather
from tests import e4m3_reference as E
from tests.test_rotary_gpu import _case, _want

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn


def _filled(pools):
    """Pools of bytes 1 and scales of 2, to see what is left alone."""
    shape = pools[0].shape
    return [torch.full(shape, 1, dtype=torch.uint8).view(F8) for _ in range(2)], \
           [torch.full(shape[:4], 2, dtype=torch.uint8) for _ in range(2)]


def _write(device, dtype, lens, Hq, Hkv, D, rotary, *, norm=False, ragged=True, layer=1, bs=16,
           pad=0, unmap=(), change=None, view=lambda x: x):
    qkv, p, cu, base, bt, pools = _case(dtype, lens, Hq, Hkv, D, bs=bs, pad=pad)
    if change is not None:
        change(qkv)
    for b, page in unmap:
        bt[b, page] = -1
    g = torch.Generator().manual_seed(9)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None
              for _ in range(2))
    (kp, vp), (ks, vs) = _filled(pools)
    d = view(qkv.to(device))
    dev = [t.to(device) for t in (kp, vp, ks, vs)]
    q_out = torch.full((d.shape[0], Hq, D), 5.0, dtype=dtype, device=device)
    args = dict(layer=layer, cu_seqlens=cu.to(device) if ragged else None,
                q_norm=None if wq is None else wq.to(device),
                k_norm=None if wk is None else wk.to(device))
    q_out = qk_norm_rope_kv(d[:, :Hq], d[:, Hq: Hq + Hkv], d[:, Hq + Hkv:], p.to(device),
                            None if rotary is None else rotary.to(device), dev[0], dev[1],
                            bt.to(device), base.to(device), q_out=q_out, k_scales=dev[2],
                            v_scales=dev[3], **args)
    # q is as without the 8 bits
    plain = torch.full_like(q_out, 5.0)
    p16 = [x.to(device) for x in pools]
    qk_norm_rope_kv(d[:, :Hq], d[:, Hq: Hq + Hkv], d[:, Hq + Hkv:], p.to(device),
                    None if rotary is None else rotary.to(device), p16[0], p16[1], bt.to(device),
                    base.to(device), q_out=plain, **args)
    assert torch.equal(q_out.cpu().view(torch.int16), plain.cpu().view(torch.int16))
    n = int(cu[-1])
    want_k, tol_k = _want(qkv[:n, Hq: Hq + Hkv], wk, 1e-6, p[:n], rotary, torch.float64)
    want_v = qkv[:n, Hq + Hkv:].double()
    if dtype == HF:
        want_v = torch.where(want_v.abs() <= 65504, want_v.clamp(-61440, 61440), want_v)
    touched = torch.zeros(ks.shape, dtype=torch.bool)
    out = [t.cpu() for t in dev]
    for b, m in enumerate(lens):
        for j in range(m):
            slot = int(base[b]) + j
            blk = int(bt[b, slot // bs])
            if blk < 0:
                continue
            t, at = int(cu[b]) + j, (blk, layer, slice(None), slot % bs)
            touched[at] = True
            v, s = E.quantised(want_v[t])
            assert torch.equal(torch.exp2(out[3][at].double() - 127), s)
            got = E.values(out[1][at], out[3][at])
            assert torch.equal(got.nan_to_num(7.0), v.nan_to_num(7.0))
            k, tol = want_k[t], tol_k[t]
            fine = k.isfinite()
            top = torch.where(fine, k.abs(), 0.0)
            at_top = top.argmax(-1, keepdim=True)
            top, off = top.amax(-1), tol.gather(-1, at_top)[..., 0].nan_to_num(0.0)
            s = torch.exp2(out[2][at].double() - 127)
            assert ((s == E.scale_of(top - off)) | (s == E.scale_of(top + off))).all()
            got = E.values(out[0][at], out[2][at])
            assert torch.equal(got.isnan(), ~fine)
            half = E.step((k.abs() + tol) / s[:, None]) / 2 * s[:, None]
            assert ((got - k).abs() <= half + tol)[fine].all()
    for x, s in ((out[0], out[2]), (out[1], out[3])):
        assert (s[~touched] == 2).all()
        assert (x.view(torch.uint8)[~touched] == 1).all()


@pytest.mark.parametrize("D,rot", [(128, 128), (64, 64), (128, 64), (32, 32), (80, 40), (16, 16),
                                   (256, 256), (128, 0)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_head_sizes(device, D, rot, layout):
    _write(device, BF, [5, 1, 18], 4, 2, D, Rotary(rot, 10000.0, layout=layout), norm=True)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("ragged", [True, False])
def test_types_and_norms(device, dtype, norm, ragged):
    _write(device, dtype, [3, 3, 3], 8, 2, 128, Rotary(128, 500000.0), norm=norm, ragged=ragged)


@pytest.mark.parametrize("lens,pad,bs", [([1], 0, 16), ([1] * 70, 0, 5), ([0, 4, 0, 0, 9, 0], 5, 1),
                                         ([700, 1, 300], 3, 32)])
def test_ragged_batches(device, lens, pad, bs):
    _write(device, BF, lens, 8, 2, 128, Rotary(128), pad=pad, bs=bs, layer=0)


def test_unmapped_pages(device):
    _write(device, BF, [30, 9], 4, 2, 64, Rotary(64), unmap=[(0, 1)])


def test_strided_views(device):
    def wide(x):
        w = torch.zeros(x.shape[0], x.shape[1] + 3, x.shape[2], dtype=x.dtype, device=x.device)
        w[:, 1: 1 + x.shape[1]] = x
        return w[:, 1: 1 + x.shape[1]]

    _write(device, BF, [7, 2], 3, 3, 128, Rotary(128), view=wide)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_extremes(device, dtype):
    """Rows of zeros, of the smallest and largest values, of magnitudes around the
    borders of the scale and of the codes, and with infinities and NaN."""
    def change(x):
        v = x[:, 6:]                                     # Hq 4, Hkv 2
        v[0] = 0.0
        v[1] = torch.finfo(dtype).max
        v[2] = torch.finfo(dtype).tiny
        v[3, 0, 0], v[3, 1, 5], v[3, 1, 6] = float("inf"), float("nan"), -float("inf")
        v[4] = torch.finfo(dtype).smallest_normal / 64   # subnormal
        v[5] = 448.0
        v[6] = 450.0
        v[7, 0] = 448.0 * 2.0 ** -9
        # half-way between codes, and what lies under the smallest one
        v[8, 0, :16] = torch.arange(16, dtype=torch.float64) * 2.0 ** -10 + 1.0 / 16
        v[8, 0, 16] = 448.0
        v[9, 0, :32] = torch.arange(32, dtype=torch.float64) * 2.0 ** -10
        v[9, 0, 33] = 448.0
        v[10] = float("nan")
        v[11, 0, 3], v[11, 1, 3] = 57344.0, 62000.0
        k = x[:, 4:6]
        k[0] = 0.0
        k[1, 0, 7] = float("inf")
        k[2] = float("nan")

    _write(device, dtype, [13], 4, 2, 64, None, change=change)


def _gather_case(dtype, lens, starts, Hkv, D, bs, seed=3, e4m3=True):
    g = torch.Generator().manual_seed(seed)
    need = [max(1, (c + n + bs - 1) // bs) for c, n in zip(starts, lens)]
    perm = torch.randperm(sum(need) + 3, generator=g).int()
    bt = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[at: at + n]
        at += n
    shape = (len(perm), 2, Hkv, bs, D)
    if e4m3:
        pools = [E.random_pool(shape, g) for _ in range(2)]
    else:
        pools = [(torch.randn(shape, generator=g).to(dtype), None) for _ in range(2)]
    return bt, pools


def _gather(device, dtype, lens, starts, Hkv, D, *, bs=16, pad=0, ragged=True, e4m3=True,
            unmap=(), given=True):
    bt, pools = _gather_case(dtype, lens, starts, Hkv, D, bs, e4m3=e4m3)
    for b, page in unmap:
        bt[b, page] = -1
    T = sum(lens) + pad
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)
    fill = 3.0 if given else 0.0
    want = [torch.full((T, Hkv, D), fill, dtype=torch.float64) for _ in range(2)]
    for w, (x, s) in zip(want, pools):
        v = x.double() if s is None else E.values(x, s)
        for b, m in enumerate(lens):
            for j in range(m):
                slot = starts[b] + j
                page = slot // bs
                blk = int(bt[b, page]) if page < bt.shape[1] else -1
                w[int(cu[b]) + j] = v[blk, 1, :, slot % bs] if blk >= 0 else 0.0
    dev = [[None if t is None else t.to(device) for t in p] for p in pools]
    outs = dict(tokens=T, dtype=dtype)
    if given:
        outs = {n: torch.full((T, Hkv, D), 3.0, dtype=dtype, device=device)
                for n in ("k_out", "v_out")}
    got = kv_gather(dev[0][0], dev[1][0], bt.to(device),
                    torch.tensor(starts, dtype=torch.int32, device=device), layer=1,
                    cu_seqlens=cu.to(device) if ragged else None, k_scales=dev[0][1],
                    v_scales=dev[1][1], **outs)
    for x, w in zip(got, want):
        assert x.dtype == dtype
        # (fp16 rounds what lies below its normal range, once)
        assert torch.equal(x.cpu().double(), w.to(dtype).double())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [128, 64, 16, 112, 256])
@pytest.mark.parametrize("e4m3", [True, False])
def test_gather(device, dtype, D, e4m3):
    _gather(device, dtype, [5, 1, 40], [0, 37, 11], 3, D, e4m3=e4m3)


@pytest.mark.parametrize("lens,starts,pad,ragged", [
    ([1], [0], 0, False), ([4, 4], [9, 0], 0, False), ([0, 3, 0], [5, 100, 2], 4, True),
    ([2] * 70, [7] * 70, 0, True), ([900], [13], 0, True)])
@pytest.mark.parametrize("given", [True, False])
def test_gather_batches(device, lens, starts, pad, ragged, given):
    _gather(device, BF, lens, starts, 8, 128, pad=pad, ragged=ragged, given=given)


@pytest.mark.parametrize("bs", [1, 5, 16, 64])
def test_gather_pages(device, bs):
    """Pages of any size, one of them not mapped."""
    _gather(device, BF, [40, 9], [3, 0], 2, 64, bs=bs, unmap=[(0, 40 // bs)])


def test_gather_of_nothing(device):
    _gather(device, BF, [0, 0], [3, 4], 2, 64)


def test_commit_moves_scales(device):
    g = torch.Generator().manual_seed(5)
    B, N, bs, D, Hkv, layers = 5, 40, 16, 64, 3, 2
    ctx = torch.tensor([3, 16, 30, 0, 17], dtype=torch.int32)
    pages = 6
    bt = torch.randperm(B * pages + 2, generator=g)[: B * pages].view(B, pages).int()
    shape = (B * pages + 2, layers, Hkv, bs, D)
    (k, ks), (v, vs) = (E.random_pool(shape, g) for _ in range(2))
    paths = torch.full((B, N), -1, dtype=torch.int32)
    path_lens = torch.tensor([1, 4, 20, 3, 2], dtype=torch.int32)
    for b in range(B):
        nodes = [0] + sorted((torch.randperm(N - 1, generator=g)[: int(path_lens[b]) - 1] + 1).tolist())
        paths[b, : len(nodes)] = torch.tensor(nodes)
    paths[4, 1] = 0                                     # not rising: refused
    want = [x.clone() for x in (k.view(torch.uint8), v.view(torch.uint8), ks, vs)]
    for w in want:
        old = w.clone()
        for b in range(4):
            for j in range(int(path_lens[b])):
                to, at = int(ctx[b]) + j, int(ctx[b]) + int(paths[b, j])
                w[bt[b, to // bs], :, :, to % bs] = old[bt[b, at // bs], :, :, at % bs]
    dev = [x.to(device) for x in (k, v, ks, vs)]
    out = kv_commit(dev[0], dev[1], bt.to(device), ctx.to(device), paths.to(device),
                    path_lens.to(device), k_scales=dev[2], v_scales=dev[3])
    assert out.status.cpu().tolist() == [0, 0, 0, 0, 1]
    for x, w in zip(dev, want):
        assert torch.equal(x.cpu().view(torch.uint8), w)


def test_cache_with_scales(device):
    """A cache of e4m3 pools: copies on write and tree commits carry the scales."""
    cfg = KVCacheConfig(num_layers=2, num_kv_heads=2, head_dim=64, total_gpu_blocks=32,
                        element_size_bytes=1)
    kv = PagedKVCache(cfg, device=device, dtype=F8)
    assert kv.key_scales.shape == kv.key_pool.shape[:4]
    g = torch.Generator().manual_seed(1)
    for pool, scales in ((kv.key_pool, kv.key_scales), (kv.value_pool, kv.value_scales)):
        codes, s = E.random_pool(pool.shape, g)
        pool.copy_(codes.to(device))
        scales.copy_(s.to(device))
    kv.register_sequence_with_prefix(1, list(range(20)))
    kv.fork_sequence(1, 2)
    kv.append_tokens(2, 1)                              # a private copy of the last page
    a, b = kv.get_block_table(1)[1], kv.get_block_table(2)[1]
    assert a != b
    for t in (kv.key_pool.view(torch.uint8), kv.value_pool.view(torch.uint8), kv.key_scales,
              kv.value_scales):
        assert torch.equal(t[a, :, :, :4], t[b, :, :, :4])
    base = torch.tensor([20], dtype=torch.int32, device=device)
    kv.append_tokens(1, 7)
    desc = kv.prepare_batch_metadata([1])
    table = desc.block_tables.clone()
    read = dict(tokens=7, k_scales=kv.key_scales, v_scales=kv.value_scales)
    before, _ = kv_gather(kv.key_pool, kv.value_pool, table, base, **read)
    path = torch.tensor([[0, 2, 6, -1, -1, -1, -1]], dtype=torch.int32, device=device)
    assert kv.commit_tree_paths([1], desc, base, path,
                                torch.tensor([3], dtype=torch.int32, device=device)) == [23]
    after, _ = kv_gather(kv.key_pool, kv.value_pool, table, base, **read)
    assert torch.equal(after[:3], before[[0, 2, 6]])


def test_captured_write_and_gather(device):
    """One graph replayed over changing inputs, next to eager work."""
    qkv, p, cu, base, bt, pools = _case(BF, [5, 12], 4, 2, 128)
    (kp, vp), (ks, vs) = _filled(pools)
    kp, vp, ks, vs, bt, base, cu, p, x = (t.to(device) for t in
                                          (kp, vp, ks, vs, bt, base, cu, p, qkv))
    rotary = Rotary(128, device=device)
    k_out, v_out = (torch.zeros(17, 2, 128, dtype=BF, device=device) for _ in range(2))

    def step(src):
        q = qk_norm_rope_kv(src[:, :4], src[:, 4:6], src[:, 6:], p, rotary, kp, vp, bt, base,
                            cu_seqlens=cu, k_scales=ks, v_scales=vs)
        kv_gather(kp, vp, bt, base, cu_seqlens=cu, k_scales=ks, v_scales=vs, k_out=k_out,
                  v_out=v_out)
        return q

    step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = step(x)
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(BF))
        graph.replay()
        got = [t.clone() for t in (q, k_out, v_out, ks, vs, kp.view(torch.uint8))]
        q2 = step(x)
        torch.cuda.synchronize()
        for a, b in zip(got, (q2, k_out, v_out, ks, vs, kp.view(torch.uint8))):
            assert torch.equal(a, b)
