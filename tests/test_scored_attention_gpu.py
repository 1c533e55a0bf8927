"""GPU tier: capped, biased and windowed attention (cfa_tree_attention_scored,
cfa_prompt_attention) against 64-bit references; tolerances are derived in
scored_reference.attend."""
import numpy as np
import pytest
import torch

from cudaforge_amd import tree as T
from cudaforge_amd.verify import (prompt_attention, prompt_attention_workspace_bytes, tree_attention,
                                  tree_attention_workspace_bytes)
from tests import scored_reference as R

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _slopes(Hq, sign=1.0):
    return torch.tensor([sign * 2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)])


def _score(name, Hq):
    """Score arguments by name: c cap, b bias, w<window>."""
    kw = {}
    for part in name.split("+"):
        if part.startswith("c"):
            kw["cap"] = float(part[1:] or 50)
        elif part == "b":
            kw["slopes"] = _slopes(Hq)
        elif part == "bneg":
            kw["slopes"] = _slopes(Hq, -0.02)
        elif part.startswith("w"):
            kw["window"] = int(part[1:])
    return kw


def _args(kw, device):
    return dict(soft_cap=kw.get("cap", 0.0), window=kw.get("window", 0),
                alibi_slopes=kw["slopes"].to(device) if "slopes" in kw else None)


def _mask_tensor(masks, device):
    return torch.from_numpy(np.array(masks, dtype=np.uint64).view(np.int64)).to(device)


def _tree(device, lens, N, Hq, Hkv, D, name, *, dtype=BF, bs=16, layers=1, layer=0, first=0,
          masks=None, seed=0, qscale=2.0, spoil=None, **call):
    q, kp, vp, bt = R.tree_case(lens, N, Hq, Hkv, D, dtype, bs=bs, layers=layers, seed=seed,
                                qscale=qscale)
    if masks is None:
        masks = [int(m) for m in T.ancestor_masks(T.binary_tree_parents(N))]
    kw = _score(name, Hq)
    q = q[:, first:].contiguous()
    want, tol = R.tree_want(q, kp, vp, bt, lens, masks, layer=layer, first=first,
                            scale=call.get("sm_scale"), **kw)
    if spoil:
        spoil(kp, vp, bt)
    got = tree_attention(q.to(device), kp.to(device), vp.to(device), bt.to(device),
                         torch.tensor(lens, dtype=torch.int32, device=device),
                         _mask_tensor(masks, device), layer=layer, first_node=first,
                         **_args(kw, device), **call)
    err = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), (err / tol).max()
    return got


SCORES = ["c50", "c30+b", "b", "w40", "c+w33", "b+w100", "c+b+w64", "c200", "c3", "bneg"]


@pytest.mark.parametrize("name", SCORES)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_scores(device, name, dtype, D):
    _tree(device, [200, 63, 1, 0], 15, 8, 2, D, name, dtype=dtype)


def test_plain_scores_in_fp16(device):
    _tree(device, [200, 63, 1, 0], 15, 8, 2, 128, "", dtype=HF)


@pytest.mark.parametrize("name", ["c50", "b", "w20", "c+b+w7"])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 4), (7, 1), (32, 8), (24, 2), (130, 1)])
def test_single_tokens(device, name, Hq, Hkv):
    """Plain decode: a tree of one node; contexts from none to several pages."""
    _tree(device, [0, 1, 15, 16, 17, 63, 64, 65, 300], 1, Hq, Hkv, 64, name)


@pytest.mark.parametrize("N", [2, 16, 17, 31, 63, 64])
@pytest.mark.parametrize("name", ["c50", "b+w50"])
def test_tree_sizes(device, N, name):
    _tree(device, [130, 5], N, 8, 2, 128, name)


def test_more_rows_than_one_block(device):
    """G * N = 8 * 63 rows: two blocks a sequence; and 16 heads a KV head."""
    _tree(device, [100, 9], 63, 8, 1, 128, "c+b")
    _tree(device, [100, 9], 40, 16, 1, 64, "c+w17")


@pytest.mark.parametrize("first", [1, 7, 14])
@pytest.mark.parametrize("name", ["c50", "b+w3", "w2"])
def test_a_level_of_the_tree(device, first, name):
    _tree(device, [100, 0], 15, 8, 2, 64, name, first=first)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 100])
@pytest.mark.parametrize("name", ["c50", "c+b", "w300", "b"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_splits(device, splits, name, dtype):
    """Ragged contexts, so that short ones leave splits without keys."""
    _tree(device, [900, 64, 0, 333], 5, 8, 2, 64, name, dtype=dtype, num_splits=splits)


def test_splits_give_the_same_sums_whatever_max_keys(device):
    a = _tree(device, [900, 64], 5, 8, 2, 64, "c+b", num_splits=4)
    b = _tree(device, [900, 64], 5, 8, 2, 64, "c+b", num_splits=4, max_keys=912)
    assert torch.equal(a, b)
    _tree(device, [900, 64], 5, 8, 2, 64, "c+b", max_keys=64)     # a guess too small


@pytest.mark.parametrize("bs", [16, 32, 48])
def test_pages_and_layers(device, bs):
    _tree(device, [100, 77], 7, 4, 2, 64, "c+w60", bs=bs, layers=3, layer=2)


def test_long_split_refills_its_page_table(device):
    """More than 16384 keys in one split: the ring of page lookups turns."""
    _tree(device, [41000, 16390], 1, 2, 1, 64, "c50", num_splits=1)
    _tree(device, [41000, 25], 2, 2, 1, 64, "b+w30000", num_splits=1)


def test_scores_beyond_the_polynomial(device):
    """Scores of several caps: the exponential form of tanh; large scales."""
    _tree(device, [200, 31], 7, 8, 2, 128, "c10", qscale=30.0)
    _tree(device, [200, 31], 7, 8, 2, 128, "c10+b", qscale=30.0, dtype=HF)
    _tree(device, [200, 31], 7, 8, 2, 128, "c30000", qscale=30.0)
    _tree(device, [200, 31], 7, 8, 2, 128, "c1000000", qscale=2.0)


def test_row_without_keys_gives_zeros(device):
    masks = [1, 0, 4 | 1, 0]                            # nodes 1 and 3 see nothing of the tree
    for name in ("c50", "b", "w1", "c+b"):
        for splits in (1, 3):
            got = _tree(device, [0, 200], 4, 8, 2, 64, name, masks=masks, num_splits=splits)
            assert (got[0, 1] == 0).all() and (got[0, 3] == 0).all()


def test_masks_of_each_sequence(device):
    chain = [int(m) for m in T.ancestor_masks(T.chain_parents(9))]
    star = [int(m) for m in T.ancestor_masks([-1] + [0] * 8)]
    for name in ("b+w5", "c+b", "w3"):
        _tree(device, [70, 20], 9, 8, 2, 64, name, masks=[chain, star])


def test_pages_in_front_of_the_window_are_not_read(device):
    """They hold NaN and infinity, or are no longer mapped."""
    def spoil(kp, vp, bt):
        # the window of 40 leaves positions 461 .. of 500 + 1, page 28 on
        for page in range(28):
            blk = int(bt[0, page])
            kp[blk] = float("nan")
            vp[blk] = float("inf")
            if page % 2:
                bt[0, page] = -1
        kp[int(bt[0, 28]), :, :, : 500 - 39 - 28 * 16] = float("nan")
        vp[int(bt[0, 28]), :, :, : 500 - 39 - 28 * 16] = float("-inf")

    for splits in (1, 2):
        for name in ("w40", "c+w40", "b+w40"):
            _tree(device, [500], 1, 8, 2, 64, name, spoil=spoil, num_splits=splits)


def test_slots_behind_the_sequence_are_not_read(device):
    def spoil(kp, vp, bt):
        blk = int(bt[0, 6])                             # slots 96 .. 111, 100 of them in use
        kp[blk, :, :, 103 - 96:] = float("nan")
        vp[blk, :, :, 103 - 96:] = float("nan")

    for name in ("c50", "b", "w9"):
        _tree(device, [100], 3, 8, 2, 128, name, spoil=spoil)


def test_nodes_behind_the_last_visible_are_not_read(device):
    """A padded batch: nodes 5 .. 8 of the first tree do not exist, their slots
    hold NaN; their queries see the context alone."""
    chain = [int(m) for m in T.ancestor_masks(T.chain_parents(9))]
    masks = [chain[:5] + [0] * 4, chain]

    def spoil(kp, vp, bt):
        for pos in range(70 + 5, 70 + 9):
            kp[int(bt[0, pos // 16]), :, :, pos % 16] = float("nan")
            vp[int(bt[0, pos // 16]), :, :, pos % 16] = float("inf")

    for name in ("c50", "b", "w9", "c+b+w3"):
        for splits in (1, 2):
            _tree(device, [70, 20], 9, 8, 2, 64, name, masks=masks, spoil=spoil, num_splits=splits)


def test_nothing_visible_reads_nothing(device):
    def spoil(kp, vp, bt):
        kp[:] = float("nan")
        vp[:] = float("nan")

    for ctx, name in ((0, "c50"), (0, "b"), (37, "w1"), (64, "b+w1")):
        got = _tree(device, [ctx], 3, 8, 2, 64, name, masks=[0, 0, 0], spoil=spoil)
        assert (got == 0).all()


def test_alignment(device):
    """q is copied where it does not begin on 16 bytes; out and pools are refused."""
    q, kp, vp, bt = R.tree_case([50], 3, 8, 2, 64, BF)
    masks = [1, 3, 5]
    want, tol = R.tree_want(q, kp, vp, bt, [50], masks, window=20)
    off = torch.zeros(q.numel() + 1, dtype=BF, device=device)
    view = off[1:].view(q.shape)
    view.copy_(q)
    a = [kp.to(device), vp.to(device), bt.to(device), torch.tensor([50], dtype=torch.int32,
                                                                  device=device)]
    m = _mask_tensor(masks, device)
    got = tree_attention(view, *a, m, window=20)
    assert ((got.cpu().double() - want).abs() <= tol).all()
    with pytest.raises(ValueError, match="aligned"):
        tree_attention(view, *a, m, window=20, out=view)
    with pytest.raises(ValueError, match="aligned"):
        pool = torch.zeros(kp.numel() + 1, dtype=BF, device=device)[1:].view(kp.shape)
        tree_attention(view, pool, *a[1:], m, window=20)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=device)
    got = prompt_attention(view[0], *a, cu, window=20)
    # (as the chain of three nodes)
    want, tol = R.prompt_want(q[0], kp, vp, bt, [50], [3], window=20)
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_out_may_be_q(device):
    """Every row is read before it is written, by the same work-group."""
    q, kp, vp, bt = (x.to(device) for x in R.tree_case([300, 40], 15, 8, 2, 64, BF))
    lens = torch.tensor([300, 40], dtype=torch.int32, device=device)
    m = _mask_tensor([int(x) for x in T.ancestor_masks(T.binary_tree_parents(15))], device)
    for splits in (1, 3):
        want = tree_attention(q, kp, vp, bt, lens, m, soft_cap=30.0, num_splits=splits)
        got = q.clone()
        tree_attention(got, kp, vp, bt, lens, m, soft_cap=30.0, num_splits=splits, out=got)
        assert torch.equal(got, want)


def test_corrupt_tables_and_lengths_stay_in_the_pool(device):
    """Block ids and lengths outside what there is are clamped."""
    q, kp, vp, bt = R.tree_case([100, 30], 3, 8, 2, 64, BF)
    bt[0, 2], bt[1, 0] = 10 ** 6, -7
    for lens in ([100, 30], [-5, 10 ** 6], [2 ** 31 - 1, -2 ** 31]):
        out = tree_attention(q.to(device), kp.to(device), vp.to(device), bt.to(device),
                             torch.tensor(lens, dtype=torch.int32, device=device),
                             _mask_tensor([1, 3, 5], device), soft_cap=50.0, max_keys=103, window=20)
        assert torch.isfinite(out).all()


# -- prompts -------------------------------------------------------------------

def _prompt(device, lens, ctx, Hq, Hkv, D, name, *, dtype=BF, bs=16, layers=1, layer=0, pad=0,
            seed=0, qscale=2.0, spoil=None, view=None, **call):
    both = [c + n for c, n in zip(ctx, lens)]
    _, kp, vp, bt = R.tree_case(both, 0, Hq, Hkv, D, dtype, bs=bs, layers=layers, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    n = sum(lens)
    q = (qscale * torch.randn(n + pad, Hq, D, generator=g)).to(dtype)
    kw = _score(name, Hq)
    want, tol = R.prompt_want(q, kp, vp, bt, ctx, lens, layer=layer, scale=call.get("sm_scale"), **kw)
    if spoil:
        spoil(kp, vp, bt)
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=device)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=device)
    qd = q.to(device) if view is None else view(q.to(device))
    got = prompt_attention(qd, kp.to(device), vp.to(device), bt.to(device),
                           torch.tensor(ctx, dtype=torch.int32, device=device), cu, layer=layer,
                           out=out, **_args(kw, device), **call)
    assert got is out
    res = got.cpu().double()
    assert (res[n:] == 7.0).all()
    assert torch.isfinite(res).all()
    err = (res[:n] - want[:n]).abs()
    assert (err <= tol[:n]).all(), (err / tol[:n]).max()
    return got


@pytest.mark.parametrize("name", SCORES + [""])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_scores(device, name, dtype, D):
    _prompt(device, [150, 1, 64, 0, 33], [0, 200, 7, 50, 300], 8, 2, D, name, dtype=dtype, pad=3)


@pytest.mark.parametrize("lens,ctx", [([1], [0]), ([2], [0]), ([63], [0]), ([64], [0]), ([65], [0]),
                                      ([257], [0]), ([300], [500]), ([1] * 9, [0] * 9),
                                      ([3] * 70, list(range(70))), ([0, 0, 5, 0], [0, 9, 9, 0])])
@pytest.mark.parametrize("name", ["c50", "b+w45"])
def test_prompt_lengths(device, lens, ctx, name):
    _prompt(device, lens, ctx, 8, 2, 64, name, pad=2)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 4), (7, 1), (12, 4), (96, 1), (130, 1), (256, 1)])
def test_prompt_heads(device, Hq, Hkv):
    _prompt(device, [70, 9], [0, 33], Hq, Hkv, 64, "c+b")


@pytest.mark.parametrize("splits", [1, 2, 5, 50])
@pytest.mark.parametrize("name", ["c50", "b", "c+b+w200"])
def test_prompt_splits(device, splits, name):
    _prompt(device, [200, 0, 31], [400, 60, 0], 8, 2, 64, name, num_splits=splits, pad=4)


@pytest.mark.parametrize("guess", [1, 16, 17, 1000])
def test_prompt_guesses_only_plan(device, guess):
    _prompt(device, [200, 31], [40, 0], 8, 2, 64, "c50", max_query=guess, max_keys=guess)


def test_prompt_pages_layers_and_strides(device):
    for bs in (16, 48):
        _prompt(device, [50, 61], [70, 0], 4, 2, 64, "b+w90", bs=bs, layers=3, layer=1)
    _prompt(device, [50, 61], [70, 0], 4, 2, 64, "c50",
            view=lambda x: x.transpose(0, 1).contiguous().transpose(0, 1))


def test_prompt_reads_no_key_behind_its_block(device):
    """Slots behind the chunk, and a window's pages in front, hold NaN."""
    def behind(kp, vp, bt):
        blk = int(bt[0, 12])                            # slots 192 .. 207, 200 in use
        kp[blk, :, :, 8:] = float("nan")
        vp[blk, :, :, 8:] = float("nan")

    def front(kp, vp, bt):
        for page in range(5):                           # the first query sees 100 - 19 = 81 on
            kp[int(bt[0, page])] = float("nan")
            vp[int(bt[0, page])] = float("nan")
            bt[0, page] = -1

    for name in ("c50", "b"):
        _prompt(device, [100], [100], 8, 2, 64, name, spoil=behind)
    _prompt(device, [100], [100], 8, 2, 64, "c+w20", spoil=front)


def test_prompt_starts_behind_row_zero(device):
    """cu_seqlens that begins behind 0: the rows in front are left alone."""
    _, kp, vp, bt = R.tree_case([40, 30], 0, 4, 2, 64, BF)
    q = torch.randn(75, 4, 64, generator=torch.Generator().manual_seed(3)).to(BF)
    want, tol = R.prompt_want(q[5:], kp, vp, bt, [0, 0], [40, 30], cap=50.0)
    for splits in (1, 2):
        out = torch.full(q.shape, 7.0, dtype=BF, device=device)
        prompt_attention(q.to(device), kp.to(device), vp.to(device), bt.to(device),
                         torch.zeros(2, dtype=torch.int32, device=device),
                         torch.tensor([5, 45, 75], dtype=torch.int32, device=device),
                         soft_cap=50.0, out=out, num_splits=splits)
        res = out.cpu().double()
        assert (res[:5] == 7.0).all()
        assert ((res[5:] - want).abs() <= tol).all()


def test_prompt_equals_tree_of_a_chain(device):
    """A chunk of 20 tokens as a prompt and as a chain-shaped tree."""
    lens = [90]
    q, kp, vp, bt = R.tree_case(lens, 20, 8, 2, 128, BF)
    qd, kd, vd, bd = (x.to(device) for x in (q, kp, vp, bt))
    ctx = torch.tensor(lens, dtype=torch.int32, device=device)
    chain = [int(m) for m in T.ancestor_masks(T.chain_parents(20))]
    for kw in (dict(soft_cap=50.0), dict(window=30), dict(soft_cap=20.0, window=11)):
        a = tree_attention(qd, kd, vd, bd, ctx, _mask_tensor(chain, device), num_splits=1, **kw)
        b = prompt_attention(qd[0], kd, vd, bd, ctx,
                             torch.tensor([0, 20], dtype=torch.int32, device=device), num_splits=1,
                             **kw)
        assert torch.equal(a[0], b)


# -- calls ----------------------------------------------------------------------

def test_streams_graphs_and_workspaces(device):
    """Captured once and replayed over growing contexts, with eager calls of the
    same shape between; the two graphs have workspaces of their own."""
    q, kp, vp, bt = R.tree_case([500, 300], 3, 8, 2, 64, BF)
    qd, kd, vd, bd = (x.to(device) for x in (q, kp, vp, bt))
    ctx = torch.tensor([10, 20], dtype=torch.int32, device=device)
    m = _mask_tensor([1, 3, 5], device)
    cu = torch.tensor([0, 3, 6], dtype=torch.int32, device=device)
    kw = dict(soft_cap=50.0, window=256, num_splits=4)

    def tree(ws=None, out=None):
        return tree_attention(qd, kd, vd, bd, ctx, m, max_keys=503, workspace=ws, out=out, **kw)

    def prompt(ws=None, out=None):
        return prompt_attention(qd.view(6, 8, 64), kd, vd, bd, ctx, cu, workspace=ws, out=out,
                                **kw)

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        tree(), prompt()
    torch.cuda.current_stream(device).wait_stream(side)
    need = max(tree_attention_workspace_bytes(2, 3, 8, 2, 64, 503, 4, scored=True, window=256),
               prompt_attention_workspace_bytes(6, 2, 8, 2, 64, 6, 512, 256, 4))
    assert need > 0
    ws = [torch.empty(need, dtype=torch.uint8, device=device) for _ in range(2)]
    outs = [torch.empty_like(qd), torch.empty(6, 8, 64, dtype=BF, device=device)]
    graphs = []
    for fn, w, o in ((tree, ws[0], outs[0]), (prompt, ws[1], outs[1])):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            fn(w, o)
        graphs.append(gr)
    for n in ([10, 20], [300, 299], [497, 0], [64, 128]):
        ctx.copy_(torch.tensor(n, dtype=torch.int32))
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], tree()) and torch.equal(outs[1], prompt())


def test_workspace_too_small_is_replaced_and_refused(device):
    import ctypes

    from cudaforge_amd import _lib

    q, kp, vp, bt = R.tree_case([500], 1, 8, 2, 64, BF)
    args = (q.to(device), kp.to(device), vp.to(device), bt.to(device),
            torch.tensor([500], dtype=torch.int32, device=device), _mask_tensor([1], device))
    small = torch.empty(16, dtype=torch.uint8, device=device)
    a = tree_attention(*args, soft_cap=50.0, num_splits=3, workspace=small)
    b = tree_attention(*args, soft_cap=50.0, num_splits=3)
    assert torch.equal(a, b)
    rc = _lib.load().cfa_tree_attention_scored(
        *(t.data_ptr() for t in args[:3]), 0, args[3].data_ptr(), args[3].shape[1],
        args[4].data_ptr(), kp.shape[0], 1, 0, 16, args[5].data_ptr(), 0, 1, 1, 0, 8, 2, 64,
        ctypes.c_float(0.125), ctypes.c_float(50.0), None, 0, 501, 3, b.data_ptr(),
        small.data_ptr(), 16, None)
    assert rc == _lib.CFA_ERR_ARG and "workspace" in _lib.last_error()


def test_refusals_on_the_device(device):
    q, kp, vp, bt = R.tree_case([50], 3, 8, 2, 64, BF)
    qd, kd, vd, bd = (x.to(device) for x in (q, kp, vp, bt))
    ctx = torch.tensor([50], dtype=torch.int32, device=device)
    m = _mask_tensor([1, 3, 5], device)
    ok = dict(q=qd, k_pool=kd, v_pool=vd, block_tables=bd, ctx_lens=ctx, tree_mask=m, soft_cap=50.0)
    tree_attention(**ok)
    for bad in (dict(q=qd.half()), dict(q=qd.float()), dict(k_pool=kd.half(), v_pool=vd.half()),
                dict(soft_cap=-1.0), dict(soft_cap=float("nan")), dict(soft_cap=float("inf")),
                dict(soft_cap=1e-9), dict(window=-1), dict(sm_scale=float("nan")),
                dict(alibi_slopes=torch.ones(7, device=device)),
                dict(alibi_slopes=torch.ones(8, device=device, dtype=BF)),
                dict(alibi_slopes=torch.ones(8)), dict(out=torch.empty(1, device=device)),
                dict(layer=1), dict(max_keys=2), dict(max_keys=10 ** 6), dict(num_splits=-1),
                dict(ctx_lens=ctx.long()), dict(tree_mask=m[:2])):
        with pytest.raises(ValueError):
            tree_attention(**{**ok, **bad})
    cu = torch.tensor([0, 3], dtype=torch.int32, device=device)
    okp = dict(q=qd[0], k_pool=kd, v_pool=vd, block_tables=bd, ctx_lens=ctx, cu_seqlens=cu)
    prompt_attention(**okp)
    for bad in (dict(q=qd), dict(q=qd[0].half()), dict(cu_seqlens=cu[:1]), dict(cu_seqlens=cu.long()),
                dict(ctx_lens=ctx.view(1, 1)), dict(block_tables=bd.repeat(2, 1)), dict(layer=-1),
                dict(max_query=0), dict(max_keys=0), dict(window=-3), dict(soft_cap=-0.5),
                dict(out=torch.empty_like(qd)), dict(num_splits=-2)):
        with pytest.raises(ValueError):
            prompt_attention(**{**okp, **bad})
    none = prompt_attention(**{**okp, "q": qd[0, :0]})
    assert none.shape == (0, 8, 64)


def test_offsets_past_32_bits(device):
    """Pages behind 2^31 elements of the pools: as from small pools."""
    Hq, Hkv, D, bs, blocks = 32, 8, 128, 16, 140000
    big = [torch.empty(blocks, 1, Hkv, bs, D, dtype=BF, device=device) for _ in range(2)]
    g = torch.Generator(device=device).manual_seed(31)
    small = [torch.randn(20, 1, Hkv, bs, D, device=device, generator=g).to(BF) for _ in range(2)]
    pages = torch.cat([torch.arange(139985, 140000), torch.arange(131071, 131076)])
    for b, s in zip(big, small):
        b[pages.to(device)] = s
    few = torch.arange(20, dtype=torch.int32, device=device).view(1, 20)
    many = pages.to(torch.int32).to(device).view(1, 20)
    q = torch.randn(1, 15, Hq, D, device=device, generator=g).to(BF)
    lens = torch.tensor([300], dtype=torch.int32, device=device)
    m = _mask_tensor([int(x) for x in T.ancestor_masks(T.binary_tree_parents(15))], device)
    cu = torch.tensor([0, 15], dtype=torch.int32, device=device)
    for kw in (dict(soft_cap=50.0), dict(window=70)):
        assert torch.equal(tree_attention(q, *big, many, lens, m, **kw),
                           tree_attention(q, *small, few, lens, m, **kw))
        assert torch.equal(prompt_attention(q[0], *big, many, lens, cu, **kw),
                           prompt_attention(q[0], *small, few, lens, cu, **kw))


def test_a_spoilt_query_spoils_its_own_row(device):
    q, kp, vp, bt = (x.to(device) for x in R.tree_case([200], 9, 8, 2, 64, BF))
    lens = torch.tensor([200], dtype=torch.int32, device=device)
    cu = torch.tensor([0, 9], dtype=torch.int32, device=device)
    m = _mask_tensor([int(x) for x in T.ancestor_masks(T.chain_parents(9))], device)
    bad = q.clone()
    bad[0, 4, 3] = float("nan")
    for kw in (dict(), dict(soft_cap=30.0), dict(alibi_slopes=_slopes(8).to(device)),
               dict(soft_cap=30.0, alibi_slopes=_slopes(8).to(device))):
        a, b = (prompt_attention(x[0], kp, vp, bt, lens, cu, **kw) for x in (q, bad))
        assert b[4, 3].isnan().all()
        b[4, 3] = a[4, 3]
        assert torch.equal(a, b)
        if kw:
            a, b = (tree_attention(x, kp, vp, bt, lens, m, **kw) for x in (q, bad))
            b[0, 4, 3] = a[0, 4, 3]
            assert torch.equal(a, b)


@pytest.mark.parametrize("B", [65, 130])
def test_many_sequences(device, B):
    """More than the 64 that a wave ranks by their length."""
    rng = np.random.default_rng(B)
    _tree(device, rng.integers(0, 150, B).tolist(), 3, 4, 2, 64, "c50")
    _tree(device, rng.integers(0, 150, B).tolist(), 1, 4, 2, 128, "b+w30")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", ["", "c50", "b", "c+b", "w20", "b+w45"])
def test_prompt_longer_than_its_table(device, name, D):
    """Tables of 48 slots: chunks and contexts that run past them see the 48, each
    token at its own position (a window that has passed them leaves nothing); a
    sequence beside them is as it would be alone."""
    cap, ctx, lens = 48, [0, 20, 300, 5], [70, 100, 9, 33]
    _, kp, vp, bt = R.tree_case([cap] * 4, 0, 8, 2, D, BF)
    assert bt.shape == (4, 3)
    q = (2.0 * torch.randn(sum(lens), 8, D, generator=torch.Generator().manual_seed(6))).to(BF)
    kw = _score(name, 8)
    at = np.concatenate([[0], np.cumsum(lens)]).tolist()
    want, tol = zip(*[R.attend(q[t: t + n], R.gather(kp, bt[b], cap, 0), R.gather(vp, bt[b], cap, 0),
                               torch.arange(c, c + n), torch.arange(cap),
                               torch.arange(c, c + n)[:, None] >= torch.arange(cap), D ** -0.5, **kw)
                      for b, (c, n, t) in enumerate(zip(ctx, lens, at))])
    for splits in (1, 2):
        got = prompt_attention(q.to(device), kp.to(device), vp.to(device), bt.to(device),
                               torch.tensor(ctx, dtype=torch.int32, device=device),
                               torch.tensor(at, dtype=torch.int32, device=device),
                               num_splits=splits, **_args(kw, device)).cpu().double()
        err = (got - torch.cat(want)).abs()
        assert (err <= torch.cat(tol)).all(), (err / torch.cat(tol)).max()


def test_prompt_lengths_out_of_range_stay_in_the_pool(device):
    q, kp, vp, bt = R.tree_case([100, 30], 20, 8, 2, 64, BF)
    qd, kd, vd, bd = (x.to(device) for x in (q, kp, vp, bt))
    for lens in ([-5, 10 ** 6], [2 ** 31 - 1, -2 ** 31], [2 ** 31 - 20, 120]):
        for kw in (dict(soft_cap=50.0), dict(window=20), dict(alibi_slopes=_slopes(8).to(device))):
            out = prompt_attention(qd.view(40, 8, 64), kd, vd, bd,
                                   torch.tensor(lens, dtype=torch.int32, device=device),
                                   torch.tensor([0, 20, 40], dtype=torch.int32, device=device), **kw)
            assert torch.isfinite(out).all()


@pytest.mark.parametrize("scored", [False, True])
def test_pages_of_2_to_the_31_elements(device, scored):
    """One page holds a whole sequence, and more elements than 32 bits count: the
    second layer's begin behind it."""
    Hq, D, bs = 4, 128, 1 << 24
    big = [torch.empty(1, 2, 1, bs, D, dtype=BF, device=device) for _ in range(2)]
    g = torch.Generator(device=device).manual_seed(17)
    small = [torch.randn(1, 2, 1, 112, D, device=device, generator=g).to(BF) for _ in range(2)]
    for b, s in zip(big, small):
        b[:, :, :, :112] = s
    table = torch.zeros(1, 1, dtype=torch.int32, device=device)
    q = torch.randn(1, 9, Hq, D, device=device, generator=g).to(BF)
    lens = torch.tensor([100], dtype=torch.int32, device=device)
    m = _mask_tensor([int(x) for x in T.ancestor_masks(T.binary_tree_parents(9))], device)
    cu = torch.tensor([0, 9], dtype=torch.int32, device=device)
    kw = dict(soft_cap=50.0) if scored else {}
    for layer in (0, 1):
        a, b = (tree_attention(q, *p, table, lens, m, layer=layer, max_keys=109, **kw)
                for p in (big, small))
        assert torch.equal(a, b)
        a, b = (prompt_attention(q[0], *p, table, lens, cu, layer=layer, max_keys=109, **kw)
                for p in (big, small))
        assert torch.equal(a, b)


@pytest.mark.parametrize("scale,cap", [(1e3, 1e-4), (1e4, 1e-6), (1e6, 1.0), (2e30, 50.0)])
@pytest.mark.parametrize("bias", [False, True])
def test_scales_far_above_the_cap(device, scale, cap, bias):
    """tanh is a step there; products of exactly 0 stay 0 (the polynomial's
    coefficients would be infinite)."""
    q, kp, vp, bt = R.tree_case([70], 3, 8, 2, 64, BF)
    q[0, 1] = 0.0
    q[0, 0, 1] = 0.0
    kw = dict(cap=cap, **(dict(slopes=_slopes(8)) if bias else {}))
    # (a product's fp32 sum may have the other sign only where |q.k| < 72 2^-24 sum |q k|)
    want, tol = R.tree_want(q, kp, vp, bt, [70], [1, 3, 5], scale=scale, **kw)
    k64 = R.gather(kp, bt[0], 73, 0)
    prod = torch.stack([q[0, :, h].double() @ k64[h // 4].t() for h in range(8)], 1)
    mag = torch.stack([q[0, :, h].double().abs() @ k64[h // 4].abs().t() for h in range(8)], 1)
    assert ((prod.abs() > 72 * 2.0 ** -24 * mag) | (mag == 0)).all()
    # the scores' error is then tanh's and exp2's alone, below 2^-20 of at most cap each
    ds = 2.0 ** -20 * (cap + 1.0) + (2.0 ** -22 * 70 if bias else 0.0)
    u = 2.0 ** -8
    A = torch.stack([(R.gather(vp, bt[0], 73, 0)[h // 4].abs()).max(0).values for h in range(8)])
    bound = u * want.abs() + 2.01 * (u + ds) * A
    got = tree_attention(q.to(device), kp.to(device), vp.to(device), bt.to(device),
                         torch.tensor([70], dtype=torch.int32, device=device),
                         _mask_tensor([1, 3, 5], device), sm_scale=scale, max_keys=73,
                         **_args(kw, device)).cpu().double()
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("scale,cap", [(1e3, 1e-4), (1e4, 1e-6), (1e6, 1.0)])
def test_zero_queries_at_scales_far_above_the_cap(device, scale, cap):
    """Every product of the call is 0, the polynomial's range: scores of 0."""
    q, kp, vp, bt = R.tree_case([70], 3, 8, 2, 64, BF)
    for kw in (dict(cap=cap), dict(cap=cap, slopes=_slopes(8))):
        want, tol = R.tree_want(q * 0, kp, vp, bt, [70], [1, 3, 5], scale=scale, **kw)
        got = tree_attention((q * 0).to(device), kp.to(device), vp.to(device), bt.to(device),
                             torch.tensor([70], dtype=torch.int32, device=device),
                             _mask_tensor([1, 3, 5], device), sm_scale=scale, max_keys=73,
                             **_args(kw, device)).cpu().double()
        assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("far", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 10 ** 15])
def test_bounds_past_32_bits(device, far):
    """A window or a guess beyond every position: as none."""
    host = R.tree_case([300], 5, 8, 2, 64, BF)
    q, kp, vp, bt = (x.to(device) for x in host)
    lens, cu = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([300], [0, 5]))
    m = _mask_tensor([int(x) for x in T.ancestor_masks(T.chain_parents(5))], device)
    kw = dict(num_splits=2, soft_cap=50.0)
    assert torch.equal(tree_attention(q, kp, vp, bt, lens, m, max_keys=305, window=far, **kw),
                       tree_attention(q, kp, vp, bt, lens, m, max_keys=305, **kw))
    assert torch.equal(prompt_attention(q[0], kp, vp, bt, lens, cu, window=far, **kw),
                       prompt_attention(q[0], kp, vp, bt, lens, cu, **kw))
    want, tol = R.prompt_want(host[0][0], *host[1:], [300], [5], cap=50.0)
    for splits in (0, 2):
        got = prompt_attention(q[0], kp, vp, bt, lens, cu, max_query=far, max_keys=far, soft_cap=50.0,
                               num_splits=splits)
        assert ((got.cpu().double() - want).abs() <= tol).all()
