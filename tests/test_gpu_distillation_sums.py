"""distill_top_logits: a reduced loss is the 64-bit sum of the rows' losses, rounded once.

With all of V logits equal and a teacher that names one class, the loss of every row is log V.  Every exponential and sum is
exact then, so a row's 64-bit loss is log V to a few 2^-53 and the sum over M rows to M of those at most (M < 2^13): within half a
step of float32, plus 2^-40 of it.  Rows that were rounded to float32 first would be off by M times their own rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [3, 6, 11, 200, 1500, 5000])
@pytest.mark.parametrize("rows", [1, 3, 32, 1000, 4096])
def test_reduced_losses_are_rounded_once(rows, cols):
    from unicorn_amd.distillation import distill_top_logits
    z = torch.zeros(rows, cols, device="cuda")
    t, i = torch.zeros(rows, 1, device="cuda"), torch.zeros(rows, 1, dtype=torch.int64, device="cuda")
    for reduction, want in (("sum", rows * math.log(cols)), ("mean", math.log(cols))):
        got = float(distill_top_logits(z, t, i, reduction=reduction))
        assert abs(got - want) <= (2.0 ** -24 + 2.0 ** -40) * want, (reduction, got, want)
