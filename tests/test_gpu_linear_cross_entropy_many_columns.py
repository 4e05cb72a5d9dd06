"""Rows of so many columns that a logit takes several runs of additions, with gradients and without: the loss, dx and
dW against the formula, with the tolerances of the operator's own tests."""
import pytest
import torch

from tests.test_gpu_linear_cross_entropy import check, make

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(1, 3, 1025), (140, 300, 1100), (33, 513, 2050), (130, 130, 16385), (70, 300, 20001), (200, 40, 33000)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_against_the_formula(gsb, dt, N, V, D, reduction):
    x, w, t = make(N, V, D, dt, seed=D, ignored=0.2 if N > 4 else 0.0)
    check(gsb, x, w, t, scale=0.9, reduction=reduction)
    gsb.check_async_errors()


@pytest.mark.parametrize("dt", DTYPES)
def test_many_rows_and_runs_of_the_depth(gsb, dt):
    """dW of 40000 rows and dx of 36000 classes: several slabs of the depth, several pieces of the vocabulary."""
    for N, V in ((40000, 70), (60, 36000)):
        x, w, t = make(N, V, 264, dt, seed=N, ignored=0.1)
        check(gsb, x, w, t, reduction="sum")
