"""Random sizes, types, views, masks and requests of the operators on learned node values, against the
formulas in 64 bits with the tolerances of their own test files."""
import numpy as np
import pytest
import torch

from tests.test_gpu_embedding import check_grad
from tests.test_gpu_linear_cross_entropy import Formula, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def log_int(rng, lo, hi):
    return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))


def view_of(rng, t):
    """The same values behind another layout: as it is, a column slice, every second row, or an odd offset."""
    rows, cols = t.shape
    how = rng.integers(0, 4)
    if how == 1:
        left, right = int(rng.integers(0, 9)), int(rng.integers(0, 9))
        big = torch.full((rows, left + cols + right), float("nan"), dtype=t.dtype, device=t.device)
        big[:, left:left + cols] = t
        return big[:, left:left + cols]
    if how == 2:
        return t.repeat_interleave(2, 0)[::2]
    if how == 3:
        off = int(rng.integers(1, 8))
        return torch.empty(rows * cols + off, dtype=t.dtype, device=t.device)[off:].view(rows, cols).copy_(t)
    return t


@pytest.mark.parametrize("seed", list(range(40)) + [206])
def test_linear_cross_entropy(gsb, seed):
    rng = np.random.default_rng(seed)
    dt = DTYPES[seed % 3]
    N, V, D = log_int(rng, 1, 2500), log_int(rng, 1, 4000), log_int(rng, 1, 300)
    scale = float(rng.choice([1.0, 0.3, -0.7]))
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(N, D, device="cuda", generator=g) * 2).to(dt)
    w = (torch.randn(V, D, device="cuda", generator=g) * D ** -0.5).to(dt)
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    t[torch.rand(N, device="cuda", generator=g) < rng.choice([0.0, 0.1, 0.9, 1.0])] = -1
    f = Formula(x, w, t, scale, dt)
    x[t < 0] = float("nan")
    need_x, need_w = [(True, True), (True, False), (False, True), (True, True)][rng.integers(0, 4)]
    xl, wl = view_of(rng, x).detach().requires_grad_(need_x), view_of(rng, w).detach().requires_grad_(need_w)
    reduction = ["none", "mean", "sum"][rng.integers(0, 3)]
    loss = gsb.ops.linear_cross_entropy(xl, wl, t, scale=scale, reduction=reduction)
    if reduction == "none":
        within(loss.detach(), f.loss, f.loss_tol, "loss")
        up = torch.randn(N, device="cuda", generator=g)
        rows = up
    else:
        up = torch.tensor(float(rng.choice([1.0, -3.0])), device="cuda")
        rows = (up / (max(1, int(f.live.sum())) if reduction == "mean" else 1)).expand(N)
    got = dict(zip([k for k, n in (("dx", need_x), ("dW", need_w)) if n],
                   torch.autograd.grad(loss, [v for v, n in ((xl, need_x), (wl, need_w)) if n], up)))
    dx, dx_tol, dw, dw_tol = f.grads(rows, dt)
    if need_x:
        within(got["dx"], dx, dx_tol, "dx %s" % ((N, V, D, dt),))
    if need_w:
        within(got["dW"], dw, dw_tol, "dW %s" % ((N, V, D, dt),))
    gsb.check_async_errors()


@pytest.mark.parametrize("seed", range(30))
def test_embedding(gsb, seed):
    rng = np.random.default_rng(1000 + seed)
    dt = DTYPES[seed % 3]
    rows, D, n = log_int(rng, 1, 300000), log_int(rng, 1, 300), log_int(rng, 1, 30000)
    scale = float(rng.choice([1.0, 0.37]))
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(rows, D, generator=g).to(dt)
    idx = (torch.rand(n, generator=g) ** int(rng.integers(1, 8)) * rows).long().clamp(max=rows - 1)
    idx[torch.rand(n, generator=g) < rng.choice([0.0, 0.2])] = -1
    grad = torch.randn(n, D, generator=g).to(dt)
    sparse = bool(rng.integers(0, 2))
    wl = view_of(rng, w.cuda()).detach().requires_grad_()
    out = gsb.ops.embedding(wl, idx.cuda(), scale=scale, sparse=sparse)
    want = torch.where((idx >= 0)[:, None], w[idx.clamp(min=0)].float() * scale, torch.zeros(())).to(dt)
    assert torch.equal(out.detach().cpu(), want)
    (dw,) = torch.autograd.grad(out, [wl], view_of(rng, grad.cuda()))
    check_grad(dw.to_dense() if sparse else dw, idx, grad, rows, scale, dt)
    gsb.check_async_errors()
