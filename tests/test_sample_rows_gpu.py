"""GPU tier: cfa_sample_rows against its definition in 64 bits, on the host.

Tokens are whole numbers and must be equal.  The kernel's weights are off by
2^-37 of the largest at most, to either side: a sum of V = 128256 by sqrt(V) 2^-37
0.58 = 1.5e-9 of the largest weight (one standard deviation), less of the whole.
A draw whose uniform (or a top-p border) lies within 1e-9 of a step of the sums
could therefore differ; `_want` finds such draws (about one in 10^4 here) and the
tests exclude them by that rule.  Probabilities: the kept weight over the kept
mass, rounded once to fp32 (2^-24) on top of sums off by 2^-29: 2^-23 of the
value."""
import numpy as np
import pytest
import torch

from cudaforge_amd.sampling import (filtered_probs, sample_rows, sample_rows_workspace_bytes)

pytestmark = pytest.mark.gpu

NEAR = 1e-9


def _want(x, us, t, k, p, m):
    """(tokens, draws that are too near a step, probabilities) of one row."""
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max)).astype(np.float64)
    probs = np.zeros(len(x))
    live = np.flatnonzero(x > -np.inf)
    if len(live) == 0:
        return np.full(len(us), -1), np.zeros(len(us), bool), probs
    by = live[np.argsort(-x[live], kind="stable")]
    border = False
    if not t > 0:
        kept, w = by[:1], np.ones(1)
    else:
        with np.errstate(under="ignore"):
            w = np.exp((x[by] - x[by[0]]) / float(t))
        n = len(by)
        if p < 1:
            c = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            n = min(n, int((c < p * w.sum()).sum()))
            # (rank 0 is kept whatever p)
            border = bool((np.abs(c[1:] / w.sum() - p) < NEAR).any()) and not _exact(w)
        if k > 0:
            n = min(n, int(k))
        if m > 0:
            n = min(n, int((w >= m).sum()))
        n = max(n, 1)
        kept, w = by[:n], w[:n]
    order = np.argsort(kept)
    kept, w = kept[order], w[order]
    upto = np.cumsum(w)
    at = np.searchsorted(upto, us * upto[-1], side="right")
    near = np.array([np.abs(upto / upto[-1] - u).min() < NEAR for u in us]) & (not _exact(w))
    last = np.flatnonzero(w > 0)[-1]
    probs[kept] = w / upto[-1]
    return kept[np.minimum(at, last)], near | border, probs


def _exact(w):
    """Weights that are powers of two: sums without any rounding."""
    f, _ = np.frexp(w)
    return bool(np.all((f == 0.5) | (w == 0)) and w[w > 0].min() > 2.0 ** -40)


def _check(device, rows, us, probs=True, workspace=None, **kw):
    R = rows.shape[0]
    dev = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    got = sample_rows(rows.to(device), us.to(device), return_probs=probs, workspace=workspace, **dev)
    tok, pr = (got[0].cpu().numpy(), got[1].cpu().numpy()) if probs else (got.cpu().numpy(), None)
    one = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    one.update(kw)
    left_out = 0
    for r in range(R):
        s = [float(np.float32(v[r] if isinstance(v, torch.Tensor) else v)) for v in
             (one["temperature"], one["top_k"], one["top_p"], one["min_p"])]
        want, near, wp = _want(rows[r].float().numpy(), us[r].double().numpy(), *s)
        left_out += int(near.sum())
        assert np.array_equal(tok[r][~near], want[~near]), (r, s, tok[r], want)
        if probs and not near.all():
            assert np.all(np.abs(pr[r] - wp) <= 2.0 ** -23 * wp + 1e-44), (r, s)
            assert np.array_equal(pr[r] > 0, wp.astype(np.float32) > 0)
    return left_out


def _rows(R, V, seed=0, sigma=2.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (sigma * torch.randn(R, V, generator=g)).to(dtype), torch.rand(R, 3, generator=g)


@pytest.mark.parametrize("V", [1, 2, 7, 63, 1000, 8191, 8192, 8193, 16385, 32000, 50257, 128256])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05),
                                dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.02),
                                dict(temperature=0.0)])
def test_sizes_and_rules(device, V, kw):
    rows, u = _rows(3, V)
    assert _check(device, rows, u, **kw) <= 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_setting_for_each_row(device, dtype):
    R, V = 48, 20011
    rows, u = _rows(R, V, seed=1, dtype=dtype)
    g = torch.Generator().manual_seed(5)

    def pick(v, dt=torch.float32):
        return torch.tensor(v, dtype=dt)[torch.randint(0, len(v), (R,), generator=g)]

    left = _check(device, rows, u, temperature=pick([0.0, -1.0, 0.05, 0.7, 1.0, 1.7, 30.0]),
                  top_k=pick([-3, 0, 1, 2, 50, 5000, 10 ** 6], torch.int32),
                  top_p=pick([0.0, 1e-6, 0.3, 0.9, 0.999, 1.0, 2.0]),
                  min_p=pick([-1.0, 0.0, 1e-5, 0.05, 0.5, 1.0]))
    assert left <= 2


@pytest.mark.parametrize("sigma", [0.0, 1e-3, 0.3, 8.0, 60.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_and_peaked_rows(device, sigma, dtype):
    """All equal (ties over many slices, more than a bin's list holds), nearly
    equal (one bin holds the row), and rows whose tail is far down."""
    rows, u = _rows(4, 40000, seed=2, sigma=sigma, dtype=dtype)
    for kw in (dict(top_k=777), dict(top_p=0.5), dict(top_p=0.9, min_p=0.3), dict(top_k=30000),
               dict(temperature=0.5, top_p=0.999)):
        _check(device, rows, u, **kw)


def test_ties_go_to_the_lower_index(device):
    rows = torch.full((2, 30000), -1.0)
    rows[0, 20000:] = 3.0                              # 10000 equal ones, in two slices
    rows[1, ::3] = 3.0
    u = torch.tensor([[0.0, 0.4999, 0.9999]] * 2)
    got = sample_rows(rows.to(device), u.to(device), top_k=4).cpu().tolist()
    assert got == [[20000, 20001, 20003], [0, 3, 9]]
    for kw in (dict(top_k=9000), dict(top_k=1), dict(top_p=0.25), dict(top_k=10001)):
        _check(device, rows, u, **kw)
    # mass in front of the kept ones stays below a half: 500 of 1000
    flat = torch.zeros(1, 1000)
    p = filtered_probs(flat.to(device), top_p=0.5).cpu()
    assert (p[0, :500] == 0.002).all() and (p[0, 500:] == 0).all()
    assert int(sample_rows(flat.to(device), torch.tensor([[0.5]], device=device), top_k=2)) == 1


def test_masked_tokens(device):
    rows, u = _rows(6, 9000, seed=3)
    rows[0, 1:] = float("-inf")
    rows[1, :] = float("-inf")                          # nothing is left
    rows[2, :8500] = float("-inf")                      # a whole slice masked
    rows[3, 100] = float("nan")
    rows[4, :] = torch.finfo(torch.float32).min         # the lowest value: all equal
    rows[5, 77] = float("inf")
    for kw in (dict(), dict(top_k=5), dict(top_p=0.7, min_p=0.1), dict(temperature=0.0)):
        _check(device, rows, u, **kw)
    tok, p = sample_rows(rows.to(device), u.to(device), return_probs=True)
    assert (tok[1] == -1).all() and (p[1] == 0).all()
    assert (tok[0] == 0).all() and (tok[5] == 77).all()
    lowest = torch.full((1, 300), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16)
    lowest[0, 7] = 1.0
    assert int(sample_rows(lowest.to(device), torch.tensor([[0.999]], device=device))) == 7


def test_extreme_temperatures_and_values(device):
    rows, u = _rows(3, 3000, seed=4)
    for t in (1e-30, 1e-6, 1e4, 1e30, 3e38):
        _check(device, rows, u, temperature=t, top_k=100)
    big = rows * 1e37
    _check(device, big, u, top_p=0.9)
    _check(device, rows * 1e-42, u, top_k=17)           # denormals: in order, equal weights


def test_uniforms_at_the_ends(device):
    rows, _ = _rows(2, 5000, seed=6)
    u = torch.tensor([[0.0, 1.0, -1.0, float("nan"), 2.0]] * 2)
    kept = (filtered_probs(rows.to(device), top_k=10) > 0).cpu()
    got = sample_rows(rows.to(device), u.to(device), top_k=10).cpu()
    for r in range(2):
        at = torch.nonzero(kept[r]).flatten().tolist()
        assert got[r].tolist() == [at[0], at[-1], at[0], at[-1], at[-1]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strides_and_alignment(device, dtype):
    base = torch.randn(6, 10007, generator=torch.Generator().manual_seed(7)).to(dtype)
    u = torch.rand(6, 2, generator=torch.Generator().manual_seed(8))
    bd, ud = base.to(device), u.to(device)
    for view in (lambda x: x, lambda x: x[:, 1:], lambda x: x[:, 3:9000], lambda x: x[::2, 8:8008],
                 lambda x: x.t().contiguous().t()):
        v = view(bd)
        rows = view(base)
        uu = u[: rows.shape[0]]
        got = sample_rows(v, ud[: rows.shape[0]], top_k=200, temperature=0.9).cpu().numpy()
        for r in range(rows.shape[0]):
            want, near, _ = _want(rows[r].float().numpy(), uu[r].double().numpy(),
                                  float(np.float32(0.9)), 200, 1.0, 0.0)
            assert np.array_equal(got[r][~near], want[~near])


def test_many_rows_and_draws(device):
    rows, _ = _rows(300, 1003, seed=9)
    u = torch.rand(300, 64, generator=torch.Generator().manual_seed(10))
    assert _check(device, rows, u, top_p=0.95) <= 20


def test_draws_follow_the_probabilities(device):
    """4096 draws of one row: each token's share within 5 standard errors."""
    rows, _ = _rows(1, 40, seed=11, sigma=1.0)
    p = filtered_probs(rows.to(device), top_p=0.9).cpu().double()[0]
    u = (torch.arange(4096).float() + 0.5) / 4096
    tok = sample_rows(rows.expand(64, 40).contiguous().to(device), u.view(64, 64).to(device),
                      top_p=0.9).cpu().flatten().long()
    share = torch.bincount(tok, minlength=40).double() / 4096
    assert ((share - p).abs() <= 1.0 / 4096 + 1e-9).all()   # equidistant uniforms


def test_results_do_not_depend_on_the_run_or_batch(device):
    rows, u = _rows(20, 128256, seed=12)
    rd, ud = rows.to(device), u.to(device)
    a, pa = sample_rows(rd, ud, top_p=0.9, return_probs=True)
    for _ in range(3):
        b, pb = sample_rows(rd, ud, top_p=0.9, return_probs=True)
        assert torch.equal(a, b) and torch.equal(pa, pb)
    c, pc = sample_rows(rd[7:8], ud[7:8], top_p=0.9, return_probs=True)
    assert torch.equal(a[7:8], c) and torch.equal(pa[7:8], pc)


def test_generator_and_streams_and_graph(device):
    rows, u = _rows(4, 33000, seed=13)
    rd, ud = rows.to(device), u.to(device)
    g1 = torch.Generator(device=device).manual_seed(3)
    g2 = torch.Generator(device=device).manual_seed(3)
    a = sample_rows(rd, generator=g1, draws=2, top_k=9)
    want = sample_rows(rd, torch.rand(4, 2, device=device, generator=g2), top_k=9)
    assert torch.equal(a, want) and a.shape == (4, 2)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        b = sample_rows(rd, ud, top_p=0.8)
    torch.cuda.current_stream(device).wait_stream(side)
    assert torch.equal(b, sample_rows(rd, ud, top_p=0.8))
    ws = torch.empty(sample_rows_workspace_bytes(4, 33000), dtype=torch.uint8, device=device)
    temp = torch.ones(4, device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, pr = sample_rows(rd, ud, temperature=temp, top_p=0.8, return_probs=True, workspace=ws)
    for step in range(4):
        rd.copy_(torch.randn(4, 33000, generator=torch.Generator().manual_seed(step)))
        ud.copy_(torch.rand(4, 3, generator=torch.Generator().manual_seed(step)))
        temp.fill_(0.5 * step)
        graph.replay()
        torch.cuda.synchronize()
        t2, p2 = sample_rows(rd, ud, temperature=temp, top_p=0.8, return_probs=True)
        assert torch.equal(tok, t2) and torch.equal(pr, p2)


def test_filtered_verification_run(device):
    """Drafts drawn from filtered rows and verified against filtered target
    rows: with equal models every draft is accepted."""
    from cudaforge_amd.verify import chain_verify

    B, K, V = 4, 3, 5000
    g = torch.Generator().manual_seed(14)
    target = (2.0 * torch.randn(B, K + 1, V, generator=g)).to(device)
    temp = torch.tensor([0.6, 0.8, 1.0, 1.2], device=device)

    def per_row(n):
        return temp.repeat_interleave(n).contiguous()

    kw = dict(top_k=50, top_p=0.9, min_p=0.02)
    tok, dp = sample_rows(target[:, :K].reshape(B * K, V), temperature=per_row(K),
                          generator=torch.Generator(device=device).manual_seed(1),
                          return_probs=True, **kw)
    tp = filtered_probs(target.view(B * (K + 1), V), temperature=per_row(K + 1), **kw)
    u = torch.rand(B, K + 1, generator=g).to(device)
    out = chain_verify(tp.view(B, K + 1, V), dp.view(B, K, V), tok.view(B, K), u,
                       input_kind="probs", mode="cpp")
    assert out.accept_len.tolist() == [K] * B
    final = out.final.long()
    assert (tp.view(B, K + 1, V)[torch.arange(B), K, final.cpu()] > 0).all()


def test_refusals_on_the_device(device):
    rows, u = _rows(4, 100)
    rd, ud = rows.to(device), u.to(device)
    sample_rows(rd, ud)
    for bad in (dict(rows=rd.double()), dict(rows=rd[0]), dict(rows=rd[:, :0]),
                dict(uniforms=ud[:3]), dict(uniforms=ud.double()), dict(uniforms=u),
                dict(draws=2), dict(uniforms=None, draws=-1), dict(uniforms=None, draws=65),
                dict(uniforms=None, draws=0), dict(temperature=-1.0),
                dict(temperature=float("nan")), dict(temperature=float("inf")),
                dict(temperature=torch.ones(3, device=device)), dict(temperature=torch.ones(4)),
                dict(top_k=2.5), dict(top_k=torch.ones(4, device=device)), dict(top_p=0.0),
                dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=1.1),
                dict(min_p=torch.ones(4, device=device).double())):
        with pytest.raises(ValueError):
            sample_rows(**{**dict(rows=rd, uniforms=ud), **bad})
    assert sample_rows(rd[:0], ud[:0]).shape == (0, 3)


def test_offsets_past_32_bits(device):
    rows, u = _rows(3, 9000, seed=41)
    far = torch.empty((1 << 31) + 20000, device=device)
    view = far.as_strided((3, 9000), ((1 << 30) + 4, 1))
    view.copy_(rows)
    want = sample_rows(rows.to(device), u.to(device), top_p=0.9, return_probs=True)
    got = sample_rows(view, u.to(device), top_p=0.9, return_probs=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype,top,zeros,each,top_k", [
    (torch.float32, 101.5, 10000, 3333, 15000), (torch.float32, 101.5, 10000, 3333, 10001),
    (torch.bfloat16, 54.0, 3000, 3000, 5000), (torch.bfloat16, 54.0, 9000, 3000, 9500),
    (torch.float16, 54.0, 3000, 3000, 5000)])
def test_zeros_beside_negative_subnormals(device, dtype, top, zeros, each, top_k):
    """The last bin holds zeros and more than a list's 8192 of the least negative
    values; the selection's borders fall between them, where -0 has a code that no
    token has.  Kept: the first top_k by value, then index."""
    least = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    x = torch.cat([torch.tensor([top]), torch.zeros(zeros // 2), torch.zeros(zeros - zeros // 2) * -1.0]
                  + [torch.full((each,), -k * least, dtype=torch.float64).float() for k in (1, 2, 3)])
    rows = torch.stack([x[torch.randperm(len(x), generator=torch.Generator().manual_seed(s))]
                        for s in (1, 2)]).to(dtype)
    assert (rows < 0).sum() == 6 * each and (rows == 0).sum() == 2 * zeros
    u = torch.tensor([[0.0, 0.5, 0.99]] * 2)
    for k in (top_k, top_k + 1, zeros, zeros + 1, zeros + 2, zeros + 1 + each, zeros + each + 2):
        # (in front of the largest, weights of e^-54 and less each: u = 0, one draw a
        # row, lies within 1e-9 of their steps; 0.5 and 0.99 of none)
        assert _check(device, rows, u, top_k=k) <= 2


@pytest.mark.parametrize("t", [1.0, 30.0, 0.01])
def test_min_p_of_one_keeps_the_largest_alone(device, t):
    """exp((x - max) / T) >= 1 for equal values only, however near the others are."""
    near = torch.tensor([0.0, -1e-12, -1e-13, -1e-14, -1e-17, -1e-30, -2.0 ** -149, 0.0])
    for scale in (1.0, t):
        rows = (near * scale)[torch.randperm(8, generator=torch.Generator().manual_seed(3))].view(1, 8)
        p = filtered_probs(rows.to(device), temperature=t, min_p=1.0).cpu()
        assert torch.equal(p, (rows == 0).float() / (rows == 0).sum())


@pytest.mark.parametrize("t", [1.0, 8.0])
@pytest.mark.parametrize("m", [0.5, 0.25, 0.1, 0.9, 0.75])
def test_min_p_border(device, t, m):
    """Values next to max + T ln(min_p), where fp32 resolves far below T: the border is
    T ln 2 2^-50 (the logarithm) and 2^-51 (sums in fp64, of at most 19) off at most,
    so values 2e-14 T from it fall on their side."""
    import decimal

    m = float(np.float32(m))
    drop = decimal.Decimal(t) * decimal.Context(prec=40).ln(decimal.Decimal(m))
    top = float(np.float32(float(-drop)))
    border = decimal.Decimal(top) + drop                # |border| < 2^-24 T: steps of 2^-48 T
    off = [s * d * t for d in (2e-14, 1e-13, 1e-12, 1e-9) for s in (1, -1)]
    vals = np.array([top] + [float(border) + o for o in off], dtype=np.float32)
    dist = [abs(decimal.Decimal(float(v)) - border) for v in vals[1:]]
    assert min(dist) > decimal.Decimal(1e-14 * t)
    want = np.array([decimal.Decimal(float(v)) >= border for v in vals])
    assert want.sum() == 5
    rows = torch.from_numpy(vals).view(1, -1)
    p = filtered_probs(rows.to(device), temperature=t, min_p=m).cpu().numpy()[0]
    assert np.array_equal(p > 0, want)
