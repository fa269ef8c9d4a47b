"""The sums over the rows (gradients of weight and bias) where there are thousands of rows for every thread that adds them: a
thread adds at most 128 rows in float32, then 64 bits take over, so the bars of test_gpu_layer_norm hold.

dy is 1.25 in the first rows, one for every chain of additions that is possible, and 0.99 * 2^-24 -- less than half a step of a
float32 between 1 and 2 -- in all others: a chain of n rows loses every one of them, n 2^-24 in all.  x is +-1 in turn,
so that h = +-1 / sqrt(1 + eps) and all terms of a column have one sign."""
import math

import pytest
import torch

from test_gpu_layer_norm import K, U

pytestmark = pytest.mark.gpu

SMALL = 0.99 * 2.0 ** -24


@pytest.mark.parametrize("rows,cols,first", [(2000, 1 << 20, 1), (256 * 128 * 2000, 4, 256 * 128)])
def test_rows_that_one_float32_sum_would_lose(rows, cols, first):
    from unicorn_amd.normalization import layer_norm
    x = torch.ones(rows, cols, device="cuda")
    x[:, 1::2] = -1.0
    dy = torch.full((rows, cols), SMALL, device="cuda")
    dy[:first] = 1.25
    small = float(torch.tensor(SMALL))                    # as float32 holds it
    w = torch.ones(cols, device="cuda", requires_grad=True)
    b = torch.zeros(cols, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(layer_norm(x, w, b), (w, b), dy)
    total = 1.25 * first + small * (rows - first)
    h = 1.0 / math.sqrt(1.0 + 1e-5)
    sign = torch.ones(cols, device="cuda", dtype=torch.float64)
    sign[1::2] = -1.0
    # the bars of test_gpu_layer_norm: B = |h| + r mean|x| = 2 h, half a step of the result
    assert float((db.double() - total).abs().max()) <= 4 * K * U * total + U * total
    assert float((dw.double() - sign * (h * total)).abs().max()) <= 4 * K * U * total * 2 * h + U * total


def test_workspace_covers_the_partial_rows():
    """a row of 2 D sums for every 128 rounds of rows, whatever their number"""
    from unicorn_amd import native
    size = native.lib().ur_layer_norm_workspace_bytes
    for rows, cols, per in ((1 << 24, 4, 128), (1 << 20, 8192, 1), (100000, 1 << 20, 1), ((1 << 31) - 1, 8, 128)):
        parts = -(-rows // (per * 128))
        assert size(rows, cols, 0, 1) >= parts * 2 * cols * 4
