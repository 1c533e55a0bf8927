"""GPU tier: adjust_logits at the sizes where it counts, lists or shares otherwise: more
biases than it searches, more tokens than it lists, and rows that share a count.
Formula and tolerances are those of test_adjust_logits_gpu.py."""
import pytest
import torch

from tests.test_adjust_logits_gpu import BF, F32, HF, _check, _random

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [255, 256, 257, 300, 5000])
@pytest.mark.parametrize("dtype,out", [(F32, None), (BF, None), (HF, None), (BF, F32), (HF, F32)])
def test_many_biases(device, K, dtype, out):
    """With repeats (the last counts), ids outside the vocabulary and listed tokens
    among them."""
    x, args = _random(2, 9001, dtype=dtype, M=2)
    g = torch.Generator().manual_seed(K)
    ids = torch.randint(-3, 9010, (2, K), generator=g, dtype=torch.int32)
    ids[:, K // 2:] = ids[:, : K - K // 2].flip(1)
    ids[:, -30:] = args["history"][:, :30]
    args["bias_tokens"], args["bias_values"] = ids, torch.randn(2, K, generator=g) * 2
    _check(device, x, out, **args)
    args["bias_tokens"], args["bias_values"] = ids[0], args["bias_values"][0]
    _check(device, x, out, **args)


@pytest.mark.parametrize("N", [3, 64])
def test_many_biases_of_trees(device, N):
    x, args = _random(2, 8200, N=N, dtype=BF, K=700, M=3)
    _check(device, x, F32, **args)


@pytest.mark.parametrize("K", [0, 200, 300])
def test_more_tokens_than_a_slice_lists(device, K):
    """Nearly every token of a slice is in the history."""
    x, args = _random(2, 9001, L=12000, K=K, M=2)
    g = torch.Generator().manual_seed(5)
    args["history"] = torch.randint(-2, 9003, (2, 12000), generator=g, dtype=torch.int32)
    args["history"][0, :9001] = torch.randperm(9001, generator=g).int()
    args["history_lens"] = torch.tensor([12000, 11111], dtype=torch.int32)
    args["prompt_lens"] = torch.tensor([5000, 0], dtype=torch.int32)
    _check(device, x, **args)


@pytest.mark.parametrize("N,B,V", [(63, 66, 1000), (64, 33, 8193), (1, 4096, 70), (5, 820, 100)])
@pytest.mark.parametrize("dtype,out", [(F32, None), (BF, F32)])
def test_rows_that_share_a_count(device, N, B, V, dtype, out):
    """16 work-groups and more for each of 256 CUs: two rows of a sequence go by one
    count, the last of an odd number by its own."""
    x, args = _random(B, V, N=N, L=9, dtype=dtype, K=2, M=3)
    _check(device, x, out, **args)


def test_a_long_history(device):
    x, args = _random(2, 9001, L=100000, few=300)
    args["history_lens"] = torch.tensor([100000, 99999], dtype=torch.int32)
    args["prompt_lens"] = torch.tensor([70001, 3], dtype=torch.int32)
    _check(device, x, **args)
