"""GPU tier: the serving operators one after another, as a decoder uses them:
prompts in two chunks, a sampled token, a draft tree that is verified and
committed, a step behind it.

Keys and values depend on a token and its position alone, and the rotary
operator's rows do not depend on their batch: whatever way the accepted tokens
took into the pages (chunks, single steps, tree nodes moved by the commit), the
slots must hold the bits that one call over the final sequences writes.
Attention is compared with 64-bit attention over those slots, with the tolerance
derived in scored_reference.attend."""
import numpy as np
import pytest
import torch

from cudaforge_amd import tree as T
from cudaforge_amd.rotary import Rotary, qk_norm_rope_kv
from cudaforge_amd.sampling import filtered_probs, sample_rows
from cudaforge_amd.verify import kv_commit, prompt_attention, tree_attention, tree_verify
from tests import scored_reference as R

pytestmark = pytest.mark.gpu

HQ, HKV, BS, V, LAYERS = 8, 2, 16, 700, 2


class _Model:
    """Tables instead of layers: a token's q, k and v rows, and logits from the
    attention's output."""

    def __init__(self, device, dtype, D, score, seed):
        g = torch.Generator().manual_seed(seed)
        self.device, self.dtype, self.D = device, dtype, D
        self.table = (2.0 * torch.randn(V, (HQ + 2 * HKV) * D, generator=g)).to(device, dtype)
        self.head = (torch.randn(HQ * D, V, generator=g) * 4.0 / (HQ * D) ** 0.5).to(device)
        self.norm = [(1.0 + 0.1 * torch.randn(D, generator=g)).to(device) for _ in range(2)]
        self.rotary = Rotary(D, theta=10000.0, device=device)
        self.score = dict(score)
        if "slopes" in score:
            self.score["slopes"] = 2.0 ** -torch.arange(1.0, HQ + 1)
        s = self.score
        self.call = dict(soft_cap=s.get("cap", 0.0), window=s.get("window", 0),
                         alibi_slopes=s["slopes"].to(device) if "slopes" in s else None)

    def write(self, tokens, positions, kp, vp, bt, base, layer, cu=None):
        qkv = self.table[tokens.long()].view(-1, HQ + 2 * HKV, self.D)
        q, k, v = qkv.split([HQ, HKV, HKV], 1)
        return qk_norm_rope_kv(q, k, v, positions, self.rotary, kp, vp, bt, base, layer=layer,
                               cu_seqlens=cu, q_norm=self.norm[0], k_norm=self.norm[1])

    def logits(self, o):
        return o.float().flatten(-2) @ self.head


def _ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("dtype,D,score", [
    (torch.bfloat16, 128, dict(cap=30.0, window=40)), (torch.float16, 64, dict(slopes=1)),
    (torch.bfloat16, 64, dict(cap=20.0, slopes=1, window=25)), (torch.float16, 128, dict())])
def test_prompt_tree_and_decode(device, dtype, D, score):
    m = _Model(device, dtype, D, score, seed=3)
    rng = np.random.default_rng(4)
    g = torch.Generator(device=device).manual_seed(5)
    lens, B, layer = [37, 3, 64], 3, 1
    N = 15
    parents = T.binary_tree_parents(N)
    masks = [int(x) for x in T.ancestor_masks(parents)]
    mask_t = T.mask_tensor(T.ancestor_masks(parents), device)
    depth = torch.from_numpy(T.depths(parents)).to(device)
    parents_t = torch.from_numpy(parents).to(device)
    seqs = [rng.integers(0, V, n).tolist() for n in lens]
    pages = (max(lens) + 40 + BS - 1) // BS
    shape = (B * pages, LAYERS, HKV, BS, D)
    kp, vp = (torch.full(shape, float("nan"), dtype=dtype, device=device) for _ in range(2))
    bt = torch.from_numpy(rng.permutation(B * pages).astype(np.int32)).view(B, pages).to(device)

    def slots(n):
        """K and V of the sequences' first n[b] slots: one call over them, in
        other pools, pages in order; the run's must be the same bits."""
        k1, v1 = torch.zeros_like(kp), torch.zeros_like(vp)
        t1 = torch.arange(B * pages, dtype=torch.int32, device=device).view(B, pages)
        flat = _ints([t for b in range(B) for t in seqs[b][: n[b]]], device)
        pos = _ints([i for b in range(B) for i in range(n[b])], device)
        m.write(flat, pos, k1, v1, t1, _ints([0] * B, device), layer,
                _ints(np.cumsum([0] + n), device))
        for b in range(B):
            for pool, one in ((kp, k1), (vp, v1)):
                assert torch.equal(R.gather(pool.cpu(), bt[b].cpu(), n[b], layer),
                                   R.gather(one.cpu(), t1[b].cpu(), n[b], layer)), b

    def near(got, want):
        assert ((got.cpu().double() - want[0]).abs() <= want[1]).all()

    # the prompts, in two chunks (the second sequence's has one of no token)
    done = [0] * B
    for part in ([20, 3, 30], [17, 0, 34]):
        cu = _ints(np.cumsum([0] + part), device)
        flat = _ints([t for b in range(B) for t in seqs[b][done[b]: done[b] + part[b]]], device)
        pos = _ints([done[b] + i for b in range(B) for i in range(part[b])], device)
        base = _ints(done, device)
        q = m.write(flat, pos, kp, vp, bt, base, layer, cu)
        o = prompt_attention(q, kp, vp, bt, base, cu, layer=layer, max_query=max(part), **m.call)
        near(o, R.prompt_want(q.cpu(), kp.cpu(), vp.cpu(), bt.cpu(), done, part, layer=layer,
                              **m.score))
        done = [d + n for d, n in zip(done, part)]
        slots(done)
        if part[1]:
            short = o[22]                               # the second sequence's last token
    last = torch.stack([o[16], short, o[50]])
    rule = dict(temperature=torch.tensor([0.7, 1.0, 1.3], device=device), top_k=60, top_p=0.95)
    root = sample_rows(m.logits(last), generator=g, **rule)[:, 0]

    for step in range(3):
        # the draft: a tree of tokens, children drawn from its nodes' filtered rows;
        # rows of noise, or (steps 1 and 2) the model's own, a level at a time
        base = _ints(done, device)
        draft = 0.5 * torch.randn(B, N, V, device=device, generator=g)
        dp = torch.zeros_like(draft)
        tokens = torch.empty(B, N, dtype=torch.int32, device=device)
        tokens[:, 0] = root
        for lo, n in ((0, 1), (1, 2), (3, 4)):
            if step:
                pos = (base[:, None] + depth[None, lo: lo + n]).to(torch.int32).reshape(-1)
                q = m.write(tokens[:, lo: lo + n].reshape(-1), pos, kp, vp, bt, base + lo, layer)
                o = tree_attention(q.view(B, n, HQ, D), kp, vp, bt, base, mask_t[: lo + n],
                                   layer=layer, first_node=lo, max_keys=max(done) + N, **m.call)
                draft[:, lo: lo + n] = m.logits(o)
            per = {**rule, "temperature": rule["temperature"].repeat_interleave(n)}
            kids, probs = sample_rows(draft[:, lo: lo + n].reshape(B * n, V), generator=g, draws=2,
                                      return_probs=True, **per)
            dp[:, lo: lo + n] = probs.view(B, n, V)
            tokens[:, 2 * lo + 1: 2 * (lo + n) + 1] = kids.view(B, 2 * n)
        per_node = {**rule, "temperature": rule["temperature"].repeat_interleave(N)}
        pos = (base[:, None] + depth[None]).to(torch.int32).reshape(-1)
        q = m.write(tokens.reshape(-1), pos, kp, vp, bt, base, layer).view(B, N, HQ, D)
        o = tree_attention(q, kp, vp, bt, base, mask_t, layer=layer, max_keys=max(done) + N, **m.call)
        near(o, R.tree_want(q.cpu(), kp.cpu(), vp.cpu(), bt.cpu(), done, masks, layer=layer,
                            **m.score))
        tp = filtered_probs(m.logits(o).view(B * N, V), **per_node).view(B, N, V)
        u = 1.0 - torch.rand(B, 4 * 3 + 2, device=device, generator=g)
        res = tree_verify(tp, dp, parents_t, tokens, u, input_kind="probs", mode="cpp")
        assert res.status.tolist() == [0] * B
        if step:  # the same filtered rows but for the attention's roundings
            assert min(res.path_len.tolist()) >= 2
        # what is emitted is what the target's filter keeps
        n_path, path = res.path_len.tolist(), res.path.tolist()
        for b in range(B):
            end = path[b][n_path[b] - 1]
            assert tp[b, end, int(res.final[b])] > 0
            for node in path[b][1: n_path[b]]:
                assert tp[b, int(parents[node]), int(tokens[b, node])] > 0
        com = kv_commit(kp, vp, bt, base, res.path, res.path_len)
        assert com.status.tolist() == [0] * B
        for b in range(B):
            seqs[b] = seqs[b][: done[b]] + [int(tokens[b, i]) for i in path[b][: n_path[b]]]
        done = com.new_ctx_lens.tolist()
        assert done == [len(s) for s in seqs]
        slots(done)
        root = res.final.to(torch.int32)

    # a single token behind it all
    base = _ints(done, device)
    q = m.write(root, base, kp, vp, bt, base, layer).view(B, 1, HQ, D)
    one = torch.ones(1, dtype=torch.int64, device=device)
    o = tree_attention(q, kp, vp, bt, base, one, layer=layer, max_keys=max(done) + 1, **m.call)
    near(o, R.tree_want(q.cpu(), kp.cpu(), vp.cpu(), bt.cpu(), done, [1], layer=layer, **m.score))
    for b in range(B):
        seqs[b].append(int(root[b]))
    slots([len(s) for s in seqs])
    # layer 0 was never written
    assert kp[:, 0].isnan().all() and vp[:, 0].isnan().all()


def test_workspaces_of_the_host_are_refused(device):
    """Its address would be written to as the device's; nothing is launched."""
    q, kp, vp, bt = (x.to(device) for x in R.tree_case([500], 3, 8, 2, 64, torch.bfloat16))
    lens, cu = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([500], [0, 3]))
    masks = torch.tensor([1, 3, 5], device=device)
    rows = torch.randn(2, 300, device=device)
    host = torch.empty(1 << 20, dtype=torch.uint8)
    strided = torch.empty(1, dtype=torch.uint8, device=device).expand(1 << 20)
    for ws in (host, strided):
        for call in (lambda: tree_attention(q, kp, vp, bt, lens, masks, max_keys=503, workspace=ws),
                     lambda: tree_attention(q, kp, vp, bt, lens, masks, soft_cap=50.0, max_keys=503,
                                            num_splits=2, workspace=ws),
                     lambda: prompt_attention(q[0], kp, vp, bt, lens, cu, num_splits=2, workspace=ws),
                     lambda: sample_rows(rows, workspace=ws),
                     lambda: filtered_probs(rows, top_k=3, workspace=ws)):
            with pytest.raises(ValueError, match="workspace"):
                call()
