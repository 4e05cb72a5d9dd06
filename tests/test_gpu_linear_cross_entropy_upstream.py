"""Upstream gradients of very different sizes, one of them not finite: dx_i is g_i times the row's own
gradient, so no row's may depend on another's."""
import pytest
import torch

from tests.test_gpu_linear_cross_entropy import Formula, make, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# dx that makes the logits again, with and without splits; dx of kept pulls; the tiled form
SIZES = [(200, 300, 64), (150, 2000, 128), (300, 47, 256), (200, 2100, 64), (200, 700, 300), (130, 2500, 300)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", SIZES)
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_a_gradient_that_is_not_finite_stays_in_its_row(gsb, dt, N, V, D, value):
    x, w, t = make(N, V, D, dt, seed=N + V, ignored=0.3)
    t[5] = 3
    up = torch.randn(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    f = Formula(x, w, t, 1.0, dt)
    finite = up.clone()
    up[5] = value
    finite[5] = 0.0
    for both in (False, True):
        xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_(both)
        loss = gsb.ops.linear_cross_entropy(xl, wl, t, reduction="none")
        dx = torch.autograd.grad(loss, [xl, wl][:1 + both], up)[0]
        want, tol, _, _ = f.grads(finite, dt)
        assert not bool(torch.isfinite(dx[5]).any())
        dx[5] = 0
        within(dx, want, tol, "dx of the other rows")
        assert not bool(dx[~f.live].any()), "rows that do not count have no gradient"


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", SIZES)
def test_rows_with_small_gradients_keep_their_digits(gsb, dt, N, V, D):
    """One row's upstream gradient is 2^40 times the others': theirs lose nothing by it."""
    x, w, t = make(N, V, D, dt, seed=N + V)
    up = torch.randn(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) * 2.0 ** 6
    f = Formula(x, w, t, 1.0, dt)
    want, tol, _, _ = f.grads(up, dt)
    up[3], want[3] = 2.0 ** 46, 0
    for both in (False, True):
        xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_(both)
        loss = gsb.ops.linear_cross_entropy(xl, wl, t, reduction="none")
        dx = torch.autograd.grad(loss, [xl, wl][:1 + both], up)[0]
        dx[3] = 0
        within(dx, want, tol, "dx")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 300])
def test_dw_of_gradients_of_different_sizes(gsb, dt, D):
    """dW row by row of the vocabulary against the formula with upstream gradients over twelve orders of two;
    a class that only small ones reach keeps its digits."""
    N, V = 260, 300
    x, w, t = make(N, V, D, dt, seed=D)
    g = torch.Generator(device="cuda").manual_seed(3)
    up = torch.randn(N, device="cuda", generator=g) * 2.0 ** -torch.randint(0, 24, (N,), device="cuda", generator=g).float()
    f = Formula(x, w, t, 1.0, dt)
    _, _, want, tol = f.grads(up, dt)
    # fp16 holds g (p - target) at 2^14 / max |g|, so a term is off by another half of its smallest step
    if dt == torch.float16:
        tol = tol + float(up.abs().max()) * 2.0 ** -39 * x.double().abs().sum(0)
    wl = w.detach().requires_grad_()
    (dw,) = torch.autograd.grad(gsb.ops.linear_cross_entropy(x, wl, t, reduction="none"), [wl], up)
    within(dw, want, tol, "dW")
