"""update_balance_bias (torch operations only) without a GPU: the comparison with the average is exact."""
import pytest
import torch

from unicorn_amd.routing import update_balance_bias


@pytest.mark.parametrize("counts", [[3, 1, 2, 2], [1, 0, 0], [0, 0, 0], [7], [33554433, 33554431], [16777217, 16777216, 16777215],
                                    [2147483647, 2147483645, 2147483646, 2147483646, 1], [999999999] * 7,
                                    [100000001] * 6 + [99999995]])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float64])
def test_every_count_is_held_against_the_average(counts, dtype):
    bias = torch.full((len(counts),), 0.25)
    got = update_balance_bias(bias, torch.tensor(counts, dtype=dtype), 0.125)
    assert got is bias
    total, n = sum(counts), len(counts)
    want = [0.25 + 0.125 * ((total > c * n) - (total < c * n)) for c in counts]
    assert bias.tolist() == want


def test_counts_of_other_types_and_gradients():
    bias = torch.zeros(3, requires_grad=True)
    update_balance_bias(bias, torch.tensor([2.5, 0.5, 1.5]), 1.0)
    assert bias.tolist() == [-1.0, 1.0, 0.0] and bias.requires_grad
