"""GPU tier: attention of few rows over e4m3 codes where keys that a row does not see,
or hardly weighs, lie in its tiles: slots that hold anything, and values far larger
than the ones that it sees."""
import pytest
import torch

from cudaforge_amd.verify import prompt_attention, tree_attention
from tests import cached_reference as C
from tests import e4m3_reference as E

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _int(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("N", [1, 2])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("ctx", [100, 96, 64, 7, 0])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_rows_that_see_nothing_are_zeros(device, N, D, splits, ctx, dtype):
    """Empty masks under a window of one: every slot from ctx on holds NaN codes and a
    scale of infinity, and where ctx begins a page that page is not mapped (its entry's
    block, the first of the pool, holds the same)."""
    pages = (ctx + N + 15) // 16
    g = torch.Generator().manual_seed(1)
    pools = [E.random_pool((pages + 2, 1, 2, 16, D), g) for _ in range(2)]
    bt = torch.arange(1, pages + 1, dtype=torch.int32)[None]
    for codes, scales in pools:
        c = codes.view(torch.uint8)
        c[0], scales[0] = 0x7f, 255
        for slot in range(ctx, pages * 16):
            c[bt[0, slot // 16], :, :, slot % 16] = 0x7f
            scales[bt[0, slot // 16], :, :, slot % 16] = 255
    if ctx % 16 == 0:
        bt[0, ctx // 16] = -1
    dev = [t.to(device) for p in pools for t in p]
    q = torch.randn(1, N, 8, D, generator=g).to(dtype).to(device)
    got = tree_attention(q, dev[0], dev[2], bt.to(device), _int([ctx], device),
                         torch.zeros(N, dtype=torch.int64, device=device), k_scales=dev[1],
                         v_scales=dev[3], window=1, num_splits=splits)
    assert (got == 0).all()


def _large_row(dtype, N, Hkv, D, spread, lens, g, at):
    """Pools whose V rows are 2^spread smaller than that of slot `at`, whose values are
    about 2^14 (2^24 in bf16)."""
    pools, bt = C.case(lens, N, Hkv, D, dtype, e4m3=True)
    top = 14 if dtype == HF else 24
    codes, scales = pools[1]
    x = torch.rand(codes.shape, generator=g) + 1.0                # 1 to 2
    x *= torch.randint(0, 2, x.shape, generator=g) * 2 - 1
    codes.copy_((x * 128.0).to(torch.float8_e4m3fn))              # 128 to 256, of 448
    scales.fill_(127 - 7 + top - spread)
    scales[bt[0, at // 16], :, :, at % 16] = 127 - 7 + top
    return pools, bt


def _near(got, want, A, dtype):
    """The output's rounding (u = eps / 2 of it; fp16's below its normal range 2^-25), and
    p's in values and sum: of 16 bits (u), and by the score's, D + 8 <= 136 fp32
    roundings (2^-24) of products whose magnitudes add up to less than 2^4."""
    u = torch.finfo(dtype).eps / 2
    tol = u * want.abs() + 2 * (u + 136 * 2.0 ** -20) * A + (2.0 ** -25 if dtype == HF else 0.0)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), (err / tol).max()


def _plain(q, pools, bt, see, n):
    """Output [rows, Hq, D] and A = sum p |v| of q's rows over the first n slots."""
    k, v = (C.rows(p, bt[0], n, 0) for p in pools)
    out, A = [], []
    G = q.shape[1] // k.shape[0]
    for h in range(q.shape[1]):
        s = q[:, h].double() @ k[h // G].t() * q.shape[2] ** -0.5
        p = torch.softmax(s.masked_fill(~see, float("-inf")), -1)
        out.append(p @ v[h // G])
        A.append(p @ v[h // G].abs())
    return torch.stack(out, 1), torch.stack(A, 1)


@pytest.mark.parametrize("spread", [14, 16, 20, 24, 28])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("ctx", [0, 40, 300])
def test_values_below_an_unseen_one(device, spread, D, dtype, ctx):
    """A tree whose root does not see its child, of few rows and, with four more nodes,
    of many: the child's V is 2^spread larger."""
    g = torch.Generator().manual_seed(spread)
    N = 6
    pools, bt = _large_row(dtype, N, 1, D, spread, [ctx], g, ctx + 1)
    q = torch.randn(1, N, 8, D, generator=g).to(dtype)
    masks = torch.tensor([1, 3, 1, 1, 1, 1])
    dev = [t.to(device) for p in pools for t in p]
    args = dict(k_scales=dev[1], v_scales=dev[3])
    see = torch.cat([torch.ones(N, ctx, dtype=torch.bool),
                     (masks[:, None] >> torch.arange(N) & 1).bool()], 1)
    want, A = _plain(q[0], pools, bt, see, ctx + N)
    for nodes in (2, N):                                         # 16 rows, 48 rows
        for splits in (0, 1, 2):
            got = tree_attention(q[:, :nodes].to(device), dev[0], dev[2], bt.to(device),
                                 _int([ctx], device), masks[:nodes].to(device),
                                 num_splits=splits, **args)
            _near(got[0], want[:nodes], A[:nodes], dtype)


@pytest.mark.parametrize("spread", [16, 20, 28])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_values_below_one_of_no_weight(device, spread, dtype):
    """The same where every row sees the large value, with a score so far below the
    others' that its share is less than 2^-50 of theirs."""
    g = torch.Generator().manual_seed(spread)
    D, ctx = 64, 70
    pools, bt = _large_row(dtype, 3, 1, D, spread, [ctx], g, 33)
    codes, scales = pools[0]
    codes.fill_(0.0)                                             # every other score 0
    codes[bt[0, 2], 0, 0, 1] = torch.full((D,), -1.0).to(torch.float8_e4m3fn)
    scales.fill_(127)
    q = torch.full((1, 2, 8, D), 8.0).to(dtype)                  # its score -64, p 2^-92
    masks = torch.tensor([1, 3])
    dev = [t.to(device) for p in pools for t in p]
    see = torch.cat([torch.ones(2, ctx, dtype=torch.bool), torch.tensor([[1, 0], [1, 1]]).bool()], 1)
    want, A = _plain(q[0], pools, bt, see, ctx + 2)
    args = dict(k_scales=dev[1], v_scales=dev[3])
    for splits in (0, 1, 2):
        got = tree_attention(q.to(device), dev[0], dev[2], bt.to(device), _int([ctx], device),
                             masks.to(device), num_splits=splits, **args)
        _near(got[0], want, A, dtype)
    # and as a prompt's chunk
    got = prompt_attention(q[0].to(device), dev[0], dev[2], bt.to(device), _int([ctx], device),
                           _int([0, 2], device), **args)
    _near(got, want, A, dtype)


@pytest.mark.parametrize("N", [1, 3, 8, 30, 63])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("splits", [1, 3])
def test_values_that_are_all_alike(device, N, D, dtype, splits):
    """Each element of V the same in every row, coded under different scales: what the
    probabilities are rounded to is in the row's sum too, so that they cancel but for fp32
    roundings (2^-24 each, of less than 2^10 of them), far less than half a step."""
    g = torch.Generator().manual_seed(N)
    pools, bt = C.case([500], N, 2, D, dtype, e4m3=True)
    codes, scales = pools[1]
    value = torch.randint(8, 16, (D,), generator=g).float() / 8        # 1 to 2, exact
    up = torch.randint(-3, 7, scales.shape, generator=g)               # 2^up is in the code
    codes.copy_((value * torch.exp2(up.float())[..., None]).to(torch.float8_e4m3fn))
    scales.copy_((127 - up).to(torch.uint8))
    q = (4.0 * torch.randn(1, N, 8, D, generator=g)).to(dtype)
    mask = torch.arange(N)
    mask = (1 << mask) | ((1 << mask) - 1)                             # a chain
    dev = [t.to(device) for p in pools for t in p]
    got = tree_attention(q.to(device), dev[0], dev[2], bt.to(device), _int([500], device),
                         mask.to(device), k_scales=dev[1], v_scales=dev[3], num_splits=splits)
    assert torch.equal(got.cpu(), value.to(dtype).expand_as(q))
