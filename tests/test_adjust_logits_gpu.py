"""GPU tier: penalties, biases and masks on logits against the formula in 64 bits.

Tolerance: one rounding to the output's type (eps / 2 of the value), behind at most
six roundings in fp32 (2^-24 each) of the logit, of the penalty's terms and of the
bias, whose magnitudes add up to `mag`: eps / 2 (|x| + 2^-21 mag) + 2^-21 mag.
fp16 rounds what lies below its normal range by 2^-25 at most, bf16 and fp32 less.
What nothing touches keeps its value, rounded once."""
import pytest
import torch

from cudaforge_amd import tree
from cudaforge_amd.sampling import adjust_logits, filtered_probs, sample_rows

pytestmark = pytest.mark.gpu

F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def _want(x, out_dtype, *, history=None, history_lens=None, prompt_lens=None, repetition=1.0,
          frequency=0.0, presence=0.0, node_tokens=None, tree_mask=None, bias_tokens=None,
          bias_values=None, allowed=None, allowed_index=None):
    B, V = x.shape[0], x.shape[-1]
    rows = x.double().reshape(B, -1, V).clone()
    mag = rows.abs()
    N = rows.shape[1]
    each = [torch.as_tensor(v, dtype=torch.float32).expand(B).double().tolist()
            for v in (repetition, frequency, presence)]
    for b in range(B):
        r, f, p = (v[b] for v in each)
        L = 0 if history is None else history.shape[1]
        n = L if history_lens is None else min(max(int(history_lens[b]), 0), L)
        at = 0 if prompt_lens is None else int(prompt_lens[b])
        toks = [] if history is None else history[b].tolist()[:n]
        seen, made = set(toks), toks[max(at, 0):]
        for i in range(N):
            mine = list(made)
            if node_tokens is not None:
                mask = int(tree_mask[b, i] if tree_mask.dim() == 2 else tree_mask[i])
                mine += [int(node_tokens[b, j]) for j in range(N) if mask >> j & 1]
            for t in seen | set(mine):
                if not 0 <= t < V:
                    continue
                v, c = float(rows[b, i, t]), mine.count(t)
                v = v / r if v > 0 else v * r
                rows[b, i, t] = v - (f * c + p if c else 0.0)
                mag[b, i, t] += abs(v) + abs(f) * c + abs(p)
        if bias_tokens is not None:
            bt = bias_tokens if bias_tokens.dim() == 1 else bias_tokens[b]
            bv = bias_values if bias_values.dim() == 1 else bias_values[b]
            for t, v in dict(zip(bt.tolist(), bv.double().tolist())).items():
                if 0 <= t < V:
                    rows[b, :, t] += v
                    mag[b, :, t] += abs(v)
    if allowed is not None:
        words = allowed.reshape(-1, allowed.shape[-1])
        for r in range(B * N):
            m = r if allowed_index is None else int(allowed_index.reshape(-1)[r])
            if not 0 <= m < words.shape[0]:
                continue
            v = torch.arange(V)
            ok = (words[m][v // 32] >> (v % 32).int()) & 1
            rows[r // N, r % N, ok == 0] = float("-inf")
    tol = 2.0 ** -21 * mag
    tol = torch.finfo(out_dtype).eps / 2 * (rows.abs() + tol) + tol
    if out_dtype == HF:
        tol = tol + 2.0 ** -25
    return rows.reshape(x.shape), tol.reshape(x.shape)


def _dev(device, args):
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in args.items()}


def _compare(got, want, tol):
    got = got.cpu().double()
    fine = want.isfinite()
    assert torch.equal(got[~fine].nan_to_num(5.0), want[~fine].nan_to_num(5.0))
    assert ((got - want).abs() <= tol)[fine].all()


def _check(device, x, out_dtype=None, view=None, **args):
    want, tol = _want(x, out_dtype or x.dtype, **args)
    d = x.to(device) if view is None else view(x.to(device))
    dev = _dev(device, args)
    got = adjust_logits(d, out_dtype=out_dtype, **dev)
    assert got.dtype == (out_dtype or x.dtype) and got.shape == x.shape
    _compare(got, want, tol)
    if out_dtype in (None, x.dtype):
        mine = d.clone() if view is None else d
        assert adjust_logits(mine, out=mine, **dev) is mine
        assert torch.equal(mine.nan_to_num(9.0), got.nan_to_num(9.0))
    return got


def _random(B, V, N=0, L=50, dtype=F32, seed=0, K=0, M=0, few=30):
    g = torch.Generator().manual_seed(seed)
    shape = (B, N, V) if N else (B, V)
    x = (torch.randn(shape, generator=g) * 3).to(dtype)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, dtype=torch.int32)

    few = ints(0, V, few)
    args = dict(history=few[ints(0, len(few), B, L).long()] if L else torch.empty(B, 0).int(),
                history_lens=ints(0, L + 1, B), prompt_lens=ints(0, L + 1, B),
                repetition=torch.rand(B, generator=g) + 0.6,
                frequency=torch.rand(B, generator=g) - 0.2, presence=torch.rand(B, generator=g))
    if N:
        args["node_tokens"] = few[ints(0, len(few), B, N).long()]
        parents = [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, N)]
        args["tree_mask"] = tree.mask_tensor(tree.ancestor_masks(parents), "cpu")
    if K:
        args["bias_tokens"] = torch.stack([torch.randperm(V, generator=g)[:K].int()
                                           for _ in range(B)])
        args["bias_values"] = torch.randn(B, K, generator=g) * 2
    if M:
        args["allowed"] = ints(-2 ** 31, 2 ** 31 - 1, M, (V + 31) // 32)
        args["allowed_index"] = ints(-1, M, *shape[:-1])
    return x, args


@pytest.mark.parametrize("dtype,out", [(F32, None), (BF, None), (HF, None), (BF, F32), (HF, F32),
                                       (F32, F32)])
@pytest.mark.parametrize("V", [1, 7, 8, 33, 1000, 4096, 4097, 20001])
def test_types_and_sizes(device, dtype, out, V):
    x, args = _random(3, V, dtype=dtype, K=min(V, 5), M=2, few=min(V, 30))
    _check(device, x, out, **args)


@pytest.mark.parametrize("N", [1, 2, 9, 63, 64])
@pytest.mark.parametrize("dtype,out", [(BF, F32), (F32, None)])
def test_trees(device, N, dtype, out):
    x, args = _random(3, 9001, N=N, dtype=dtype, K=3, M=3)
    _check(device, x, out, **args)


@pytest.mark.parametrize("B,L", [(1, 0), (1, 1), (70, 3), (2, 5000)])
def test_histories(device, B, L):
    x, args = _random(B, 5000, L=L)
    _check(device, x, **args)


def test_each_alone(device):
    x, args = _random(4, 3001, L=40, K=9, M=2)
    hist = {k: args[k] for k in ("history", "history_lens", "prompt_lens")}
    _check(device, x)
    _check(device, x, **hist)                            # nothing to do: as they are
    _check(device, x, history=args["history"], repetition=1.3)
    _check(device, x, frequency=0.5, **hist)
    _check(device, x, presence=-0.25, **hist)
    _check(device, x, bias_tokens=args["bias_tokens"], bias_values=args["bias_values"])
    _check(device, x, bias_tokens=args["bias_tokens"][0], bias_values=args["bias_values"][0])
    _check(device, x, allowed=args["allowed"], allowed_index=args["allowed_index"])
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (4, 94), dtype=torch.int32,
                          generator=torch.Generator().manual_seed(2))
    _check(device, x, allowed=words)


def test_untouched_values_keep_their_bits(device):
    x, args = _random(2, 5000, dtype=BF)
    got = adjust_logits(x.to(device), **_dev(device, args)).cpu()
    hit = torch.zeros(x.shape, dtype=torch.bool)
    hit.scatter_(1, args["history"].long(), True)
    assert torch.equal(got[~hit].view(torch.int16), x[~hit].view(torch.int16))


def test_ids_outside_the_vocabulary_and_the_same_twice(device):
    x, args = _random(2, 500, L=8, N=4)
    args["history"][0] = torch.tensor([-1, 500, 2 ** 31 - 1, -2 ** 31, 3, 3, 3, 499])
    args["history_lens"] = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32)
    args["prompt_lens"] = torch.tensor([5, -7], dtype=torch.int32)
    args["node_tokens"][0] = torch.tensor([-1, 3, 3, 700])
    args["bias_tokens"] = torch.tensor([9, -1, 9, 800, 9, 3], dtype=torch.int32)
    args["bias_values"] = torch.tensor([5.0, 1.0, 6.0, 1.0, -2.0, 0.5])
    _check(device, x, **args)


def test_masks_leave_nothing(device):
    """Rows of masked tokens alone, bits behind the vocabulary, indexes of no mask."""
    x, _ = _random(4, 77)
    allowed = torch.zeros(2, 3, dtype=torch.int32)
    allowed[1] = -1
    index = torch.tensor([0, 1, -1, 2], dtype=torch.int32)
    got = _check(device, x, allowed=allowed, allowed_index=index).cpu()
    assert (got[0] == float("-inf")).all() and torch.equal(got[1:], x[1:])


def test_infinities_and_nan(device):
    """-inf stays, a masked NaN or +inf is gone, an untouched NaN stays."""
    x, _ = _random(2, 64)
    x[:, 3], x[:, 4], x[:, 5], x[:, 40] = -float("inf"), float("inf"), float("nan"), float("nan")
    hist = torch.tensor([[3, 4, 5], [3, 4, 6]], dtype=torch.int32)
    allowed = torch.full((2, 2), -1, dtype=torch.int32)
    allowed[1, 0] &= ~(1 << 4 | 1 << 5)
    got = _check(device, x, history=hist, repetition=1.5, frequency=0.25, presence=1.0,
                 allowed=allowed).cpu()
    assert (got[:, 3] == -float("inf")).all()
    assert got[0, 4] == float("inf") and got[1, 4] == -float("inf")
    assert got[0, 5].isnan() and got[1, 5] == -float("inf") and got[:, 40].isnan().all()


def test_strided_and_unaligned_rows(device):
    def wide(x):                              # rows of a wider buffer, at an odd element
        w = torch.zeros(*x.shape[:-1], x.shape[-1] + 5, dtype=x.dtype, device=x.device)
        w[..., 3: 3 + x.shape[-1]] = x
        return w[..., 3: 3 + x.shape[-1]]

    for dtype in (BF, F32):
        x, args = _random(3, 5003, N=3, dtype=dtype, M=2)
        _check(device, x, view=wide, **args)
    x, args = _random(3, 5003, dtype=HF, M=2)
    _check(device, x, view=wide, **args)
    # every node's row from one: logits [B, 1, V] expanded
    x, args = _random(2, 3001, N=5, dtype=BF)
    one = x[:, :1].expand(2, 5, 3001)
    want, tol = _want(one.contiguous(), BF, **args)
    d = x.to(device)
    _compare(adjust_logits(d[:, :1].expand(2, 5, 3001), **_dev(device, args)), want, tol)
    # transposed: copied first
    x, args = _random(6, 300)
    want, tol = _want(x, F32, **args)
    _compare(adjust_logits(x.t().contiguous().to(device).t(), **_dev(device, args)), want, tol)


def test_out_elsewhere(device):
    x, args = _random(3, 2000, dtype=BF)
    want, tol = _want(x, F32, **args)
    out = torch.full((3, 2100), 7.0, device=device)
    got = adjust_logits(x.to(device), out=out[:, 50:2050], **_dev(device, args))
    _compare(got, want, tol)
    assert (out[:, :50] == 7.0).all() and (out[:, 2050:] == 7.0).all()


def test_one_chain_is_a_tree_of_one_path(device):
    """Row i of a chain counts the drafts in front of it."""
    B, K, V = 3, 4, 700
    x, args = _random(B, V, N=K + 1)
    g = torch.Generator().manual_seed(4)
    drafts = torch.randint(0, 5, (B, K), dtype=torch.int32, generator=g)
    args["node_tokens"] = torch.cat([torch.full((B, 1), -1, dtype=torch.int32), drafts], 1)
    args["tree_mask"] = tree.mask_tensor(tree.ancestor_masks([-1, 0, 1, 2, 3]), "cpu")
    got = _check(device, x, **args)
    hist = args["history"]
    for i in range(K + 1):
        rows = []
        for b in range(B):
            n = int(args["history_lens"][b])
            rows.append(torch.cat([hist[b, :n], drafts[b, :i]]))
        for b in range(B):
            p = args["prompt_lens"][b: b + 1].clamp(max=int(args["history_lens"][b]))
            alone = adjust_logits(
                x[b: b + 1, i].to(device), history=rows[b][None].to(device),
                prompt_lens=p.to(device),
                **{k: args[k][b: b + 1].to(device) for k in ("repetition", "frequency", "presence")})
            assert torch.equal(alone[0], got[b, i])


def test_in_front_of_the_sampler(device):
    """A run of the two: a grammar that leaves one token is what is drawn."""
    x, args = _random(5, 4003, dtype=BF, M=0)
    pick = torch.tensor([0, 4002, 17, 32, 31])
    allowed = torch.zeros(5, 126, dtype=torch.int32)
    for r, t in enumerate(pick.tolist()):
        allowed[r, t // 32] = -2 ** 31 if t % 32 == 31 else 1 << (t % 32)
    y = adjust_logits(x.to(device), allowed=allowed.to(device), **_dev(device, args))
    assert sample_rows(y, draws=3).cpu().long().tolist() == [[t] * 3 for t in pick.tolist()]
    p = filtered_probs(y).cpu()
    assert torch.equal(p.argmax(-1), pick) and (p.sum(-1) == 1.0).all()


def test_captured(device):
    x, args = _random(4, 9000, N=6, dtype=BF, K=4, M=3)
    dev = _dev(device, args)
    d = x.to(device)
    out = torch.empty(x.shape, device=device)
    adjust_logits(d, out=out, **dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adjust_logits(d, out=out, **dev)
    for seed in range(4):
        y, more = _random(4, 9000, N=6, dtype=BF, K=4, M=3, seed=seed)
        d.copy_(y)
        for k, v in more.items():
            dev[k].copy_(v)
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, adjust_logits(d, out_dtype=F32, **dev))
        _compare(got, *_want(y, F32, **more))


def test_on_another_stream(device):
    x, args = _random(8, 30000, dtype=BF)
    d, dev = x.to(device), _dev(device, args)
    want = adjust_logits(d, **dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = adjust_logits(d, **dev)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_offsets_past_32_bits(device):
    """Rows that begin more than 2^31 elements into their buffer."""
    V, far = 4099, 2 ** 31 + 64
    buf = torch.zeros(far + V, dtype=BF, device=device)
    x, args = _random(2, V, dtype=BF)
    view = buf.as_strided((2, V), (far, 1))
    view.copy_(x)
    _compare(adjust_logits(view, **_dev(device, args)), *_want(x, BF, **args))
    adjust_logits(view, out=view, **_dev(device, args))
    _compare(view, *_want(x, BF, **args))


def test_refusals(device):
    x = torch.zeros(2, 3, 40, device=device)
    i = torch.zeros(2, 3, dtype=torch.int32, device=device)
    m = torch.ones(3, dtype=torch.int64, device=device)

    def bad(match, logits=x, **kw):
        with pytest.raises((ValueError, TypeError), match=match):
            adjust_logits(logits, **kw)

    bad("device tensor", logits=x.cpu())
    bad("float32", logits=x.double())
    bad("V > 0", logits=x[..., :0])
    bad("V\\]", logits=x[0, 0])
    bad("history must", history=i[:1])
    bad("int32", history=i.long())
    bad("go with history", history_lens=i[:, 0])
    bad("history_lens must", history=i, history_lens=i)
    bad("positive", repetition=0.0)
    bad("positive", repetition=float("nan"))
    bad("finite", frequency=float("inf"))
    bad("presence must", presence=torch.zeros(3, device=device))
    bad("go together", node_tokens=i)
    bad("tree_mask must", node_tokens=i, tree_mask=m[:2])
    bad("at most 64", logits=torch.zeros(1, 65, 8, device=device),
        node_tokens=torch.zeros(1, 65, dtype=torch.int32, device=device),
        tree_mask=torch.ones(65, dtype=torch.int64, device=device))
    bad("go together", bias_tokens=i)
    bad("bias_tokens and bias_values must", bias_tokens=i, bias_values=torch.zeros(3, device=device))
    bad("allowed_index goes", allowed_index=i)
    bad("mask for each row", allowed=torch.zeros(2, 2, dtype=torch.int32, device=device))
    bad("allowed must be", allowed=torch.zeros(2, 1, dtype=torch.int32, device=device),
        allowed_index=i)
    bad("out_dtype", out_dtype=BF)
    bad("out must be float32", out=torch.zeros(2, 3, 40, dtype=BF, device=device))
    bad("logits' shape", out=torch.zeros(2, 40, device=device))
    bad("rows must not overlap", out=torch.zeros(1, 1, 40, device=device).expand(2, 3, 40))
    wide = torch.zeros(2, 3, 48, device=device)
    bad("not overlap", logits=wide[..., :40], out=wide[..., 4:44])
    empty = adjust_logits(torch.zeros(0, 9, device=device))
    assert empty.shape == (0, 9)
    assert adjust_logits(torch.zeros(2, 0, 9, device=device)).shape == (2, 0, 9)
