"""Classes that are masked through one column of the table (the lowest finite value or minus infinity there,
a one in x): the loss, dW and -- for a finite mask, 0 * inf being NaN in any form of it -- dx are those of the
table without these classes, and the masked rows of dW are zeros, whatever ignored rows hold."""
import pytest
import torch

from tests.test_gpu_linear_cross_entropy import Formula, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# streamed forms with and without kept pulls, fp32's, and the tiled form; rows that end inside a tile
SIZES = [(70, 60, 40), (300, 300, 64), (129, 257, 128), (200, 2500, 64), (130, 2100, 200), (140, 300, 300), (64, 2300, 300)]


def masked_inputs(N, V, D, dt, mask, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, D, device="cuda", generator=g).to(dt)
    w = (torch.randn(V, D, device="cuda", generator=g) * D ** -0.5).to(dt)
    x[:, D - 1] = 1.0
    gone = torch.rand(V, device="cuda", generator=g) < 0.3
    gone[0], gone[V - 1] = True, True
    w[gone, D - 1] = mask
    kept = (~gone).nonzero().flatten()
    t = kept[torch.randint(0, len(kept), (N,), device="cuda", generator=g)]
    t[torch.rand(N, device="cuda", generator=g) < 0.2] = -1
    t[0], t[1] = -1, -1
    return x, w, t, gone, kept


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", SIZES)
@pytest.mark.parametrize("mask", ["lowest", "-inf"])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_masked_classes(gsb, dt, N, V, D, mask, reduction):
    value = torch.finfo(dt).min if mask == "lowest" else -float("inf")
    x, w, t, gone, kept = masked_inputs(N, V, D, dt, value, N + V)
    place = torch.full((V,), -1, dtype=torch.int64, device="cuda")
    place[kept] = torch.arange(len(kept), device="cuda")
    f = Formula(x, w[kept], torch.where(t >= 0, place[t.clamp(min=0)], t), 1.0, dt)
    # ignored rows that meet the mask with other values than a one, and one that is not finite
    dead = (t < 0).nonzero().flatten()
    x[dead[::2], D - 1] = 0.0
    x[dead[1]] = float("nan")
    xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = gsb.ops.linear_cross_entropy(xl, wl, t, reduction=reduction)
    count = max(1, int(f.live.sum()))
    if reduction == "none":
        within(loss.detach(), f.loss, f.loss_tol, "loss")
        up, g = torch.ones_like(loss), torch.ones(N, device="cuda")
    else:
        within(loss.detach(), f.loss.sum() / count, f.loss_tol.sum() / count + 2.0 ** -22 * f.loss.sum() / count, "mean loss")
        up, g = torch.ones((), device="cuda"), torch.full((N,), 1.0 / count, device="cuda")
    dx, dw = torch.autograd.grad(loss, [xl, wl], up)
    want_dx, tol_dx, want_dw, tol_dw = f.grads(g, dt)
    assert not bool(dw[gone].any()), "masked classes have no gradient"
    within(dw[kept], want_dw, tol_dw, "dW")
    assert not bool(dx[dead].any())
    if mask == "lowest":
        within(dx, want_dx, tol_dx, "dx")
    with torch.no_grad():
        scores = gsb.ops.linear_cross_entropy(x, w, t, reduction="none")
    within(scores, f.loss, f.loss_tol, "loss without gradients")
    gsb.check_async_errors()


@pytest.mark.parametrize("D", [64, 100, 200])
def test_values_near_the_largest_of_fp32(gsb, D):
    """Finite values above the largest bf16 that a product leaves out: x holds them where the table is zero,
    and the table where x is."""
    g = torch.Generator(device="cuda").manual_seed(D)
    x = torch.randn(150, D, device="cuda", generator=g)
    w = torch.randn(400, D, device="cuda", generator=g) * D ** -0.5
    x[:, 3], w[:, 3] = 0.0, 0.0
    x[:, 5], w[:, 5] = 0.0, 0.0
    t = torch.randint(0, 400, (150,), device="cuda", generator=g)
    want = gsb.ops.linear_cross_entropy(x, w, t, reduction="none")
    assert bool(torch.isfinite(want).all())
    big = torch.finfo(torch.float32).max
    x[::3, 3], x[1::3, 3] = big, -big
    w[::2, 5], w[1::2, 5] = -big, 3.397e38
    assert torch.equal(gsb.ops.linear_cross_entropy(x, w, t, reduction="none"), want)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 200, 300])
def test_an_infinite_value_of_x_is_its_own_rows_alone(gsb, dt, D):
    g = torch.Generator(device="cuda").manual_seed(D)
    x = torch.randn(200, D, device="cuda", generator=g).to(dt)
    w = (torch.randn(300, D, device="cuda", generator=g).abs() * D ** -0.5).to(dt)
    t = torch.randint(0, 300, (200,), device="cuda", generator=g)
    want = gsb.ops.linear_cross_entropy(x, w, t, reduction="none")
    x[7, 2] = float("inf")
    got = gsb.ops.linear_cross_entropy(x, w, t, reduction="none")
    others = torch.arange(200, device="cuda") != 7
    assert not bool(torch.isfinite(got[7])) and torch.equal(got[others], want[others])
