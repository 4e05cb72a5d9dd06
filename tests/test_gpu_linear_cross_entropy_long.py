"""Long sums of one sign.  All logits are zero (x and the table meet in no column), so every p is a power of two
and exact, and what is left are the additions into the accumulators: each may lose a unit in the last
place of the running sum (u = 2^-23), and at most 1024 of them follow one another before the sum moves
on (fp32: 64 of the six products' high one; bf16 up to 256 columns 8192, a quarter of its half step), however
long the sum; then 32-bit sums of these, rounded to nearest, a few roundings more (16 u), and half a step of
the type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def last(v, tol, dt):
    return tol + torch.finfo(dt).eps / 2 * (v.abs() + tol) + (2.0 ** -25 if dt == torch.float16 else 0)


def bound(dt, terms, magnitude, D):
    # additions of 16 products each
    run = 64 if dt == torch.float32 else 8192 if dt == torch.bfloat16 and D <= 256 else 1024
    return (run + terms / (16 * run) / 2 + 16) * U * magnitude


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(40000, 262144, 64), (40000, 262144, 128), (20000, 262144, 256), (300, 262144, 300), (40000, 1048576, 64)])
def test_dx_of_a_large_vocabulary(gsb, dt, N, V, D):
    """dx_i = g (mean of the table's rows - w_t), about as large as the table's values."""
    if dt == torch.float32:
        N = N // 2
    g = torch.Generator(device="cuda").manual_seed(1)
    w = (torch.rand(V, D, device="cuda", generator=g) + 1).to(dt)
    w[:, 0] = 0
    x = torch.zeros(N, D, dtype=dt, device="cuda")
    x[:, 0] = 1
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    w[t] = 0.25 * w[t]                       # the targets' own rows do not cancel the sum
    xl = x.requires_grad_()
    loss = gsb.ops.linear_cross_entropy(xl, w, t, reduction="none")
    (dx,) = torch.autograd.grad(loss, [xl], torch.ones(N, device="cuda"))
    mean = w.double().mean(0)
    want = mean - w[t].double() * 1.0
    tol = last(want, bound(dt, V, mean, D) + 4 * U * w[t].double().abs(), dt)
    err = (dx.double() - want).abs()
    assert bool((err <= tol).all()), "%g over, largest error %g" % (float((err - tol).max()), float(err.max()))
    gsb.check_async_errors()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(250000, 65536, 64), (250000, 65536, 128), (250000, 32768, 256), (1000000, 128, 300), (1000000, 512, 100)])
def test_dw_of_many_rows(gsb, dt, N, V, D):
    """dW_j = sum_i g (1 / V - [t_i = j]) x_i, N / V as large as x for a class that is nobody's target."""
    if dt == torch.float32:
        N = N // 4
    g = torch.Generator(device="cuda").manual_seed(2)
    x = (torch.rand(N, D, device="cuda", generator=g) + 1).to(dt)
    x[:, 0] = 0
    w = torch.zeros(V, D, dtype=dt, device="cuda")
    w[:, 0] = 1
    t = torch.randint(0, V // 2, (N,), device="cuda", generator=g)     # the upper half: nobody's
    wl = w.requires_grad_()
    up = torch.full((), 64.0, device="cuda")
    (dw,) = torch.autograd.grad(gsb.ops.linear_cross_entropy(x, wl, t), [wl], up)
    each = 64.0 / N
    want = x.double().sum(0, keepdim=True) * each / V
    got = dw[V // 2:].double()
    # 64 / N is rounded once; g p at 2^14 is a power of two
    tol = last(want, bound(dt, N, want, D) + 4 * U * want, dt)
    err = (got - want).abs()
    assert bool((err <= tol).all()), "%g over, largest error %g of %g" % (float((err - tol).max()), float(err.max()), float(want.max()))
    gsb.check_async_errors()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [4000, 20001, 65536])
def test_logits_of_many_columns(gsb, dt, D):
    """One logit is a sum of D products of one sign and the others are zero: the loss is the logit, nearly."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.rand(130, D, device="cuda", generator=g) + 1).to(dt)
    w = torch.zeros(20, D, dtype=dt, device="cuda")
    w[3] = (torch.rand(D, device="cuda", generator=g) + 1).to(dt)
    t = torch.full((130,), 5, device="cuda")
    scale = 16.0 / D
    loss = gsb.ops.linear_cross_entropy(x, w, t, scale=scale, reduction="none")
    l = scale * (x.double() @ w.double().T)
    want = torch.logsumexp(l, 1) - l[:, 5]
    tol = bound(dt, D, l[:, 3].abs(), D) + U * (64 + 8 * l.abs().amax(1))
    err = (loss.double() - want).abs()
    assert bool((err <= tol).all()), "%g over, largest error %g" % (float((err - tol).max()), float(err.max()))
