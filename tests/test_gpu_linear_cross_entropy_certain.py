"""Rows whose target is all but certain (1 - p_t below 2^-26): every other class together is less than half a unit in
the last place of the sum, so the row's log-sum-exp is its target's logit and 1 - p_t is zero in 32 bits.  The
gradients must be as small as that: the logits are exact in 32 bits (small multiples of a power of two, as in the
tests of likely targets), so p_t may be off by one rounding of the exponential, u / 2 = 2^-24, and no more.
  dx_i  |g| (u / 2 |w_t| + sum_{j != t} 2 p_ij |w_j|)     dW_j  sum_i |g| (u / 2 [t_i = j] + 2 p_ij) |x_i|
(the twice stands for every relative error of the other classes' tiny p), and half the type's smallest step."""
import pytest
import torch

from tests.test_gpu_linear_cross_entropy import Formula, make, within
from tests.test_gpu_linear_cross_entropy_confident import rows_with, table

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(40, 5, 64), (300, 47, 64), (200, 300, 128), (60, 1999, 64), (100, 2500, 64), (80, 47, 256), (130, 300, 300), (64, 700, 520)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_no_gradient_is_left(gsb, dt, N, V, D, sign):
    w = table(V, D, V + D)
    gen = torch.Generator(device="cuda").manual_seed(N)
    t = torch.randint(0, V, (N,), device="cuda", generator=gen)
    # x = k w_t with k that the type holds and that leaves the others 2^-26 together
    x = torch.empty(N, D, dtype=torch.float64, device="cuda")
    for i, c in enumerate(t.tolist()):
        l = w @ w[c]
        for k in torch.arange(32, 64, device="cuda").double() / 8:
            others = k * l
            others[c] = -float("inf")
            if float(torch.logsumexp(others, 0) - k * l[c]) < -18.1:
                break
        else:
            raise AssertionError("the table has no such row")
        x[i] = w[c] * k
    if sign < 0:
        x = -x
    xl, wl = x.to(dt).requires_grad_(), w.to(dt).requires_grad_()
    assert torch.equal(xl.detach().double(), x) and torch.equal(wl.detach().double(), w), "the type holds the values"
    up = 1024.0
    loss = gsb.ops.linear_cross_entropy(xl, wl, t, scale=sign, reduction="sum")
    dx, dw = torch.autograd.grad(loss, [xl, wl], torch.tensor(up, device="cuda"))
    l = sign * x @ w.T
    p = torch.exp(l - torch.logsumexp(l, 1)[:, None])
    hot = torch.zeros_like(p)
    hot[torch.arange(N), t] = 1
    p = p * (1 - hot)
    assert float(p.sum(1).max()) < 2.0 ** -26
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    bound_x = up * (U / 2 * w[t].abs() + 2 * p @ w.abs()) + tiny
    bound_w = up * ((U / 2 * hot + 2 * p).T @ x.abs()) + tiny
    worst = lambda got, bound: float((got.double().abs() / bound.clamp(min=1e-300)).max())
    assert worst(dx, bound_x) <= 1 and worst(dw, bound_w) <= 1, (worst(dx, bound_x), worst(dw, bound_w))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V,D", [(47, 64), (1999, 128), (3000, 64), (300, 256), (700, 300)])
def test_small_losses_keep_their_digits(gsb, dt, V, D):
    """loss = log(1 + others / target's own): its relative error is that of the other classes' sum, r =
    u (8 max |l| + V / 16 + 64), and a few roundings, however small it is."""
    w = table(V, D, V)
    miss = [0.5, 0.1, 1e-2, 1e-3, 1e-4, 1e-6, 1e-8, 1e-10] * 4
    t = torch.randint(0, V, (len(miss),), generator=torch.Generator().manual_seed(D)).cuda()
    x = rows_with(w, t, miss)
    l = x @ w.T
    others = l.clone()
    others[torch.arange(len(t)), t] = -float("inf")
    want = torch.nn.functional.softplus(torch.logsumexp(others, 1) - l[torch.arange(len(t)), t], threshold=100)
    r = U * (8 * l.abs().amax(1) + V / 16 + 64 + 8)
    assert float(want.min()) < 1e-6
    for grad in (False, True):
        loss = gsb.ops.linear_cross_entropy(x.to(dt).requires_grad_(grad), w.to(dt), t, reduction="none").detach().double()
        assert bool(((loss - want).abs() <= r * want).all()), float(((loss - want).abs() / want / r).max())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(200, 300, 64), (90, 2500, 128), (150, 47, 256), (100, 300, 300)])
def test_gradients_without_the_losses(gsb, dt, N, V, D):
    """The plain entry has no losses to go by and makes the targets' logits once more: within the formula's bounds."""
    x, w, t = make(N, V, D, dt, seed=V, ignored=0.2)
    f = Formula(x, w, t, -0.7, dt)
    ops = torch.ops.gs_ops
    loss, lse2, pull = ops._CAPI_LinearCrossEntropy(x, w, t, -0.7, -1, True)
    up = torch.randn(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    dx, dw = ops._CAPI_LinearCrossEntropyGrad(x, w, t, lse2, pull, up, None, -0.7, -1, True, True)
    want_dx, tol_dx, want_dw, tol_dw = f.grads(up, dt)
    within(loss, f.loss, f.loss_tol, "loss")
    within(dx, want_dx, tol_dx, "dx")
    within(dw, want_dw, tol_dw, "dW")


def test_losses_that_the_caller_changes(gsb):
    """The rows' losses are the caller's: changed in place, the gradients are those of what they became."""
    x, w, t = make(60, 50, 32, torch.float32, seed=2)
    weights = torch.rand(60, device="cuda")
    grads = []
    for in_place in (False, True):
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = gsb.ops.linear_cross_entropy(xl, wl, t, reduction="none")
        loss = loss.mul_(weights) if in_place else loss * weights
        grads.append(torch.autograd.grad(loss.sum(), [xl, wl]))
    for a, b in zip(*grads):
        assert torch.equal(a, b)
