"""GPU tier: attention over caches of e4m3 codes, and through a window with first
tokens that stay visible, against 64-bit references of the values that the codes
stand for; tolerances are derived in scored_reference.attend.  (In fp16 a key or
value below 2^-14 is rounded once more, by 2^-25 at most: under the absolute 2^-20
that a score may be off by, and one part in 2^5 of the `tiny` term per key.)"""
import numpy as np
import pytest
import torch

from cudaforge_amd import tree as T
from cudaforge_amd.verify import prompt_attention, tree_attention
from tests import cached_reference as C

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _score(name, Hq):
    """Arguments by name: c<cap>, b (bias), w<window>, s<sinks>."""
    kw = {}
    for part in filter(None, name.split("+")):
        if part == "b":
            kw["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)])
        else:
            key = dict(c="cap", w="window", s="sinks")[part[0]]
            kw[key] = float(part[1:]) if key == "cap" else int(part[1:])
    return kw


def _args(kw, pools, device):
    return dict(soft_cap=kw.get("cap", 0.0), window=kw.get("window", 0), sinks=kw.get("sinks", 0),
                alibi_slopes=kw["slopes"].to(device) if "slopes" in kw else None,
                **{n: None if p[1] is None else p[1].to(device)
                   for n, p in zip(("k_scales", "v_scales"), pools)})


def _masks(N, device):
    masks = [int(m) for m in T.ancestor_masks(T.binary_tree_parents(N))]
    return masks, torch.from_numpy(np.array(masks, dtype=np.uint64).view(np.int64)).to(device)


def _int(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _close(got, want, tol):
    err = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), (err / tol).max()


def _tree(device, lens, N, Hq, Hkv, D, name, *, dtype=BF, e4m3=True, bs=16, layers=1, layer=0,
          first=0, spoil=None, **call):
    g = torch.Generator().manual_seed(7)
    pools, bt = C.case(lens, N, Hkv, D, dtype, e4m3=e4m3, bs=bs, layers=layers)
    q = (2.0 * torch.randn(len(lens), N - first, Hq, D, generator=g)).to(dtype)
    masks, mask = _masks(N, device)
    kw = _score(name, Hq)
    want, tol = C.tree_want(q, pools, bt, lens, masks, layer=layer, first=first, **kw)
    if spoil:
        spoil(pools, bt)
    got = tree_attention(q.to(device), pools[0][0].to(device), pools[1][0].to(device),
                         bt.to(device), _int(lens, device), mask, layer=layer, first_node=first,
                         **_args(kw, pools, device), **call)
    _close(got, want, tol)
    return got


def _prompt(device, lens, ctx, Hq, Hkv, D, name, *, dtype=BF, e4m3=True, bs=16, layers=1, layer=0,
            pad=0, spoil=None, **call):
    g = torch.Generator().manual_seed(8)
    pools, bt = C.case(ctx, lens, Hkv, D, dtype, e4m3=e4m3, bs=bs, layers=layers)
    q = (2.0 * torch.randn(sum(lens) + pad, Hq, D, generator=g)).to(dtype)
    kw = _score(name, Hq)
    want, tol = C.prompt_want(q, pools, bt, ctx, lens, layer=layer, **kw)
    if spoil:
        spoil(pools, bt)
    out = torch.full_like(q, 3.0).to(device)
    cu = [0] + list(np.cumsum(lens))
    got = prompt_attention(q.to(device), pools[0][0].to(device), pools[1][0].to(device),
                           bt.to(device), _int(ctx, device), _int(cu, device), layer=layer, out=out,
                           **_args(kw, pools, device), **call)
    assert got is out and (out[sum(lens):] == 3.0).all()
    _close(got[: sum(lens)], want[: sum(lens)], tol[: sum(lens)])
    return got


SCORES = ["", "c50", "c200", "b", "c30+b", "w40", "w33+s3", "c+w33+s70".replace("c+", "c50+"),
          "b+w20+s64", "c9+b+w64+s1"]


@pytest.mark.parametrize("name", SCORES)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_scores(device, name, dtype, D):
    _tree(device, [200, 63, 1, 0], 15, 8, 2, D, name, dtype=dtype)


@pytest.mark.parametrize("name", ["w33+s3", "c50+w33+s70", "b+w20+s64", "c9+b+w64+s1", "w1+s1"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_first_tokens_over_16_bits(device, name, dtype, D):
    _tree(device, [300, 63, 1, 0], 15, 8, 2, D, name, dtype=dtype, e4m3=False)
    _prompt(device, [70, 1, 33], [0, 400, 64], 8, 2, D, name, dtype=dtype, e4m3=False, pad=2)


@pytest.mark.parametrize("name", ["", "c50", "b", "w20+s5"])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 4), (7, 1), (32, 8), (24, 2), (130, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_single_tokens(device, name, Hq, Hkv, D):
    """Plain decode, contexts from none to several pages."""
    _tree(device, [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 300, 700], 1, Hq, Hkv, D, name)


@pytest.mark.parametrize("N", [2, 3, 4, 5, 16, 17, 31, 63, 64])
@pytest.mark.parametrize("name", ["", "b+w50+s9"])
def test_tree_sizes(device, N, name):
    _tree(device, [130, 5], N, 8, 2, 128, name)


def test_more_rows_than_one_block(device):
    _tree(device, [100, 9], 63, 8, 1, 128, "c50+b")
    _tree(device, [100, 9], 40, 16, 1, 64, "c50+w17+s20")


@pytest.mark.parametrize("first", [1, 7, 14])
@pytest.mark.parametrize("name", ["", "b+w3+s2", "w2+s33"])
def test_a_level_of_the_tree(device, first, name):
    _tree(device, [100, 0], 15, 8, 2, 64, name, first=first)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 100])
@pytest.mark.parametrize("name", ["", "c50+b", "w300+s100", "b", "c50+w5+s200"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_splits(device, splits, name, dtype):
    """Ragged contexts, so that short ones leave splits without keys."""
    for N, D in ((5, 64), (1, 128)):
        _tree(device, [900, 64, 0, 333], N, 8, 2, D, name, dtype=dtype, num_splits=splits)
    _prompt(device, [40, 3], [800, 0], 8, 2, 64, name, dtype=dtype, num_splits=splits)


@pytest.mark.parametrize("name", ["", "c50", "b", "w500+s30"])
def test_steps_of_the_rings(device, name):
    """Contexts of every number of tiles up to past the rings' turns."""
    for N in (1, 20):
        _tree(device, [64 * n + 7 for n in range(12)], N, 8, 2, 128, name, num_splits=1)


@pytest.mark.parametrize("bs", [16, 32, 48])
def test_pages_and_layers(device, bs):
    _tree(device, [100, 77], 7, 4, 2, 64, "c50+w60+s20", bs=bs, layers=3, layer=2)
    _tree(device, [100, 77], 1, 4, 2, 128, "", bs=bs, layers=3, layer=2)
    _prompt(device, [100, 20], [9, 77], 4, 2, 128, "w60+s20", bs=bs, layers=3, layer=1)


def test_long_split_refills_its_page_table(device):
    _tree(device, [41000, 16390], 1, 2, 1, 64, "c50", num_splits=1)
    _tree(device, [41000, 25], 5, 8, 1, 64, "b+w30000+s500", num_splits=1)


@pytest.mark.parametrize("lens,ctx", [([1], [0]), ([64], [0]), ([65, 1, 130], [0, 7, 500]),
                                      ([0, 5, 0, 300], [9, 0, 3, 100])])
@pytest.mark.parametrize("name", ["", "c50", "b+w50+s10", "w70+s100"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompts(device, lens, ctx, name, dtype):
    for D in (64, 128):
        _prompt(device, lens, ctx, 8, 2, D, name, dtype=dtype, pad=3)


def test_long_prompt(device):
    _prompt(device, [700], [0], 32, 8, 128, "")
    _prompt(device, [700], [100], 4, 1, 64, "c50+w100+s17")


@pytest.mark.parametrize("sinks,window", [(1, 1), (16, 16), (64, 64), (63, 65), (65, 63), (128, 1),
                                          (200, 40), (1000, 7), (79, 80)])
@pytest.mark.parametrize("e4m3", [True, False])
def test_borders_of_the_first_tokens(device, sinks, window, e4m3):
    """First tokens that end inside a page, a tile, at the window, and past it; pages
    between them and the window are gone, their table entries far out of the pool."""
    name = f"w{window}+s{sinks}"
    lens = [300, 143, 144, 145, 64]

    def spoil(pools, bt):
        for b, ctx in enumerate(lens):
            lo, hi = -(-sinks // 16), max(ctx - window + 1, 0) // 16
            bt[b, lo: max(hi, lo)] = 2 ** 31 - 1

    _tree(device, lens, 1, 8, 2, 128, name, e4m3=e4m3, spoil=spoil)
    _tree(device, lens, 7, 8, 2, 64, name, e4m3=e4m3)
    _prompt(device, [150, 3], [0, 200], 8, 2, 64, name, e4m3=e4m3)


def test_hidden_slots_may_hold_anything(device):
    """Codes of NaN and any scale byte behind the sequences, between the first tokens
    and the window, and in pages of others."""
    lens = [300, 20, 0]

    def spoil(pools, bt):
        for codes, scales in pools:
            c = codes.view(torch.uint8)
            used = torch.zeros(scales.shape, dtype=torch.bool)
            for b, ctx in enumerate(lens):
                for s in list(range(min(ctx, 5))) + list(range(max(0, ctx - 29), ctx + 1)):
                    used[bt[b, s // 16], :, :, s % 16] = True
            c[~used] = 0x7f
            scales[~used] = 255

    _tree(device, lens, 1, 8, 2, 128, "w30+s5", spoil=spoil)
    _tree(device, lens, 1, 8, 2, 64, "b+w30+s5", spoil=spoil, num_splits=3)


def test_nothing_visible(device):
    """A window in front of which only first tokens are left: a node that its own mask
    does not hold sees those, and without any it gets zeros."""
    pools, bt = C.case([100], 2, 2, 64, BF, e4m3=True)
    q = torch.randn(1, 2, 8, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    want, tol = C.tree_want(q, pools, bt, [100], [0, 0], window=1, sinks=3)
    dev = [t.to(device) for p in pools for t in p]
    args = dict(k_scales=dev[1], v_scales=dev[3], window=1)
    zero = torch.zeros(2, dtype=torch.int64, device=device)
    for sinks in (3, 0):
        got = tree_attention(q.to(device), dev[0], dev[2], bt.to(device), _int([100], device), zero,
                             sinks=sinks, **args)
        if sinks:
            _close(got, want, tol)
        else:
            assert (got == 0).all()


def test_values_of_very_different_sizes(device):
    """Rows of V from 2^-60 to 2^60, the large ones hardly seen; zero scales' rows."""
    for dtype, span in ((BF, 60), (HF, 12)):
        for N in (1, 9):
            def spoil(pools, bt):
                pass
            pools, bt = C.case([500], N, 1, 128, dtype, e4m3=True)
            g = torch.Generator().manual_seed(2)
            s = pools[1][1]
            s.copy_((127 - 8 + torch.randint(-span, span // 2, s.shape, generator=g)).to(torch.uint8))
            if dtype == HF:
                s.clamp_(min=127 - 14, max=127 + 5)
            q = (6.0 * torch.randn(1, N, 4, 128, generator=g)).to(dtype)
            masks, mask = _masks(N, device)
            want, tol = C.tree_want(q, pools, bt, [500], masks)
            dev = [t.to(device) for p in pools for t in p]
            got = tree_attention(q.to(device), dev[0], dev[2], bt.to(device), _int([500], device),
                                 mask, k_scales=dev[1], v_scales=dev[3])
            _close(got, want, tol)


def test_equal_to_the_cache_read_back(device):
    """Over codes as over the 16-bit cache that kv_gather makes of them."""
    from cudaforge_amd.verify import kv_gather

    for dtype in (BF, HF):
        pools, bt = C.case([300], 30, 2, 128, dtype, e4m3=True)
        q = torch.randn(1, 30, 8, 128, generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
        _, mask = _masks(30, device)
        dev = [t.to(device) for p in pools for t in p]
        lens = _int([300], device)
        got = tree_attention(q, dev[0], dev[2], bt.to(device), lens, mask, k_scales=dev[1],
                             v_scales=dev[3], soft_cap=200.0)
        n = bt.shape[1] * 16
        k, v = kv_gather(dev[0], dev[2], bt.to(device), _int([0], device), tokens=n,
                         k_scales=dev[1], v_scales=dev[3], dtype=dtype)
        pages = [x.view(-1, 16, 2, 128).transpose(1, 2).unsqueeze(1).contiguous() for x in (k, v)]
        ident = torch.arange(bt.shape[1], dtype=torch.int32, device=device)[None]
        same = tree_attention(q, *pages, ident, lens, mask, soft_cap=200.0)
        err = (got.double() - same.double()).abs().max()
        assert err <= 4 * torch.finfo(dtype).eps * same.abs().max()


def test_streams_and_graphs(device):
    """A captured call and an eager one in turn, each with its own workspace, over
    changing caches; another stream gives the same."""
    lens = [700, 33, 150]
    for N in (1, 12):
        pools, bt = C.case(lens, N, 2, 128, BF, e4m3=True)
        dev = [t.to(device) for p in pools for t in p]
        _, mask = _masks(N, device)
        q = torch.randn(3, N, 8, 128, device=device).to(BF)
        out = torch.empty_like(q)
        args = dict(k_scales=dev[1], v_scales=dev[3], window=200, sinks=4, max_keys=700 + N,
                    num_splits=3)
        btd, ctx = bt.to(device), _int(lens, device)

        def call(**kw):
            return tree_attention(q, dev[0], dev[2], btd, ctx, mask, **args, **kw)

        want = call()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = call()
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(want, other)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(out=out)
        for i in range(4):
            dev[1].copy_(torch.randint(118, 126, dev[1].shape).to(torch.uint8))
            q.copy_(torch.randn(q.shape))
            graph.replay()
            got = out.clone()
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_offsets_past_32_bits(device):
    """Pages whose codes lie past 2^32 bytes."""
    nblk, Hkv, D = 2 ** 32 // (16 * 128 * 2) + 40, 2, 128
    small, bt = C.case([90, 40], 1, Hkv, D, BF, e4m3=True)
    q = torch.randn(2, 1, 8, D, generator=torch.Generator().manual_seed(3)).to(BF)
    masks, mask = _masks(1, device)
    want, tol = C.tree_want(q, small, bt, [90, 40], masks)
    far = nblk - small[0][0].shape[0]
    dev = []
    for codes, scales in small:
        pool = torch.zeros(nblk, 1, Hkv, 16, D, dtype=torch.uint8, device=device)
        pool[far:] = codes.view(torch.uint8).to(device)
        sc = torch.zeros(nblk, 1, Hkv, 16, dtype=torch.uint8, device=device)
        sc[far:] = scales.to(device)
        dev += [pool.view(torch.float8_e4m3fn), sc]
    table = torch.where(bt >= 0, bt + far, bt).int().to(device)
    for kw in (dict(), dict(window=50, sinks=3)):
        if kw:
            want, tol = C.tree_want(q, small, bt, [90, 40], masks, **kw)
        got = tree_attention(q.to(device), dev[0], dev[2], table, _int([90, 40], device), mask,
                             k_scales=dev[1], v_scales=dev[3], **kw)
        _close(got, want, tol)


def test_corrupt_tables_stay_in_the_pool(device):
    """Block ids out of range are read as some page of the pool; nothing faults."""
    pools, bt = C.case([300, 90], 3, 2, 64, BF, e4m3=True)
    dev = [t.to(device) for p in pools for t in p]
    _, mask = _masks(3, device)
    bad = torch.full_like(bt, 2 ** 31 - 1)
    bad[1] = -(2 ** 31)
    for table, lens in ((bad, [300, 90]), (bt, [2 ** 31 - 1, -7])):
        for kw in (dict(), dict(window=20, sinks=40), dict(window=1, sinks=2 ** 31 - 1)):
            got = tree_attention(torch.ones(2, 3, 4, 64, dtype=BF, device=device), dev[0], dev[2],
                                 table.to(device), _int(lens, device), mask, max_keys=303,
                                 k_scales=dev[1], v_scales=dev[3], **kw)
            torch.cuda.synchronize()
            assert got.shape == (2, 3, 4, 64)


def test_refusals_on_the_device(device):
    pools, bt = C.case([30], 1, 2, 64, BF, e4m3=True)
    k, ks, v, vs = (t.to(device) for p in pools for t in p)
    q = torch.zeros(1, 1, 4, 64, dtype=BF, device=device)
    _, mask = _masks(1, device)
    btd, ctx, cu = bt.to(device), _int([30], device), _int([0, 1], device)

    def bad(match, k=k, v=v, **kw):
        for call in (lambda: tree_attention(q, k, v, btd, ctx, mask, **kw),
                     lambda: prompt_attention(q[0], k, v, btd, ctx, cu, **kw)):
            with pytest.raises(ValueError, match=match):
                call()

    bad("go together", k_scales=ks)
    bad("bfloat16")
    bad("float8", k=k.view(torch.uint8), v=v.view(torch.uint8), k_scales=ks, v_scales=vs)
    bad("uint8", k_scales=ks.to(torch.int32), v_scales=vs)
    bad("contiguous", k_scales=ks[..., :8], v_scales=vs)
    bad("contiguous", k_scales=ks.transpose(1, 2), v_scales=vs)
    bad("sinks", k_scales=ks, v_scales=vs, sinks=-1)
