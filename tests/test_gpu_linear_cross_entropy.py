"""Vocabulary cross entropy and its gradients against the formula in 64 bits.

Tolerances, for the inputs as they are (already rounded to their type).  u = 2^-23 bounds the
relative error of one 32-bit addition, truncated or rounded, and of one product.
  logit   a_ij = (D + 4) u |s| sum_d |x_id w_jd|      D products added in 32 bits, the scale and base change
  lse     b_i  = max_j a_ij + u (V / 16 + 64 + 4 max_j |l_ij|)   sums of V terms in runs of 16 or more
                 at a time (one addition of the running sum each), exp and log at a few units
  p_ij    relative r_ij = a_ij + b_i + 8 u, plus half a step h of the type where the matrix units
          take p in 16 bits; fp16 holds it scaled by at least 2^7, its smallest step is 2^-24: q = 2^-31
  dx_i    |g_i s| (sum_j (p_ij (r_ij + h + V u) + q) |w_jd| + 4 u |w_td|), then half a step of the type
  dW_j    sum_i |g_i s| ((p_ij (r_ij + h) + q + [t_i = j] (h + u) + N u (p_ij + [t_i = j])) |x_id|), likewise
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def make(N, V, D, dt, seed=0, ignored=0.0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(N, D, device="cuda", generator=g) * spread).to(dt)
    w = (torch.randn(V, D, device="cuda", generator=g) * D ** -0.5).to(dt)
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    t[torch.rand(N, device="cuda", generator=g) < ignored] = -1
    return x, w, t


class Formula(object):
    def __init__(self, x, w, t, scale, dt):
        V, D = w.shape
        N = x.shape[0]
        self.live = (t >= 0) & (t < V)
        X = torch.where(self.live[:, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
        W = w.double()
        l = scale * X @ W.T
        a = (D + 4) * U * abs(scale) * (X.abs() @ W.abs().T)
        lse = torch.logsumexp(l, 1)
        self.b = a.amax(1) + U * (V / 16 + 64 + 4 * l.abs().amax(1))
        tt = t.clamp(0, V - 1)
        hot = torch.zeros(N, V, dtype=torch.float64, device=x.device)
        hot[torch.arange(N, device=x.device), tt] = 1.0
        self.loss = torch.where(self.live, lse - l.gather(1, tt[:, None])[:, 0], torch.zeros_like(lse))
        self.loss_tol = self.b + a.gather(1, tt[:, None])[:, 0] + 4 * U * self.loss.abs()
        h = 0.0 if dt == torch.float32 else half_step(dt)
        q = 2.0 ** -31 if dt == torch.float16 else 0.0
        p = torch.exp(l - lse[:, None])
        r = a + self.b[:, None] + 8 * U
        self.unit_dx = scale * ((p - hot) @ W)
        self.unit_dx_tol = abs(scale) * ((p * (r + h + V * U) + q) @ W.abs() + 4 * U * hot @ W.abs())
        self.X, self.p, self.hot, self.scale = X, p, hot, scale
        self.cell_tol = p * (r + h) + q + hot * (h + U) + N * U * (p + hot)

    def grads(self, g, dt):
        g = torch.where(self.live, g.double(), torch.zeros((), dtype=torch.float64, device=g.device))
        dx, dx_tol = g[:, None] * self.unit_dx, g.abs()[:, None] * self.unit_dx_tol
        gs = g * self.scale
        dw = (self.p - self.hot).T @ (gs[:, None] * self.X)
        dw_tol = self.cell_tol.T @ (gs[:, None] * self.X).abs()
        last = lambda v, e: e + half_step(dt) * (v.abs() + e) + (2.0 ** -25 if dt == torch.float16 else 0) + 4 * U * v.abs()
        return dx, last(dx, dx_tol), dw, last(dw, dw_tol)


def within(got, want, tol, what):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), "%s: %g over the tolerance, largest error %g" % (
        what, float((err - tol).max()), float(err.max()))


def check(gsb, x, w, t, scale=1.0, reduction="mean", up=None):
    dt = x.dtype
    xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = gsb.ops.linear_cross_entropy(xl, wl, t, scale=scale, reduction=reduction)
    assert loss.dtype == torch.float32
    f = Formula(x.detach(), w.detach(), t, scale, dt)
    count = max(1, int(f.live.sum()))
    if reduction == "none":
        within(loss.detach(), f.loss, f.loss_tol, "loss")
        up = torch.ones_like(loss) if up is None else up
        g = up
    else:
        div = count if reduction == "mean" else 1
        up = torch.tensor(1.0 if up is None else up, device="cuda")
        within(loss.detach(), f.loss.sum() / div, f.loss_tol[f.live].sum() / div + 2 * U * f.loss.sum().abs() / div, "loss")
        g = (up / div).expand(t.shape[0])
    dx, dw = torch.autograd.grad(loss, [xl, wl], up)
    assert dx.dtype == dt and dw.dtype == dt and dx.shape == x.shape and dw.shape == w.shape
    want_dx, tol_dx, want_dw, tol_dw = f.grads(g, dt)
    within(dx, want_dx, tol_dx, "dx")
    within(dw, want_dw, tol_dw, "dW")
    assert not bool(dx[~f.live].any())
    return loss.detach(), dx, dw


SIZES = [(1, 1, 1), (1, 2, 16), (3, 47, 24), (1, 1000, 128), (2, 129, 64), (127, 128, 100), (128, 257, 128), (129, 255, 65),
         (130, 300, 256), (257, 1000, 33), (300, 47, 200), (513, 2000, 128), (700, 3, 256), (64, 4099, 72), (40, 700, 300),
         (300, 2500, 64), (257, 3001, 128), (130, 2100, 256), (700, 5000, 100), (120, 2049, 16), (90, 2300, 120),
         (2100, 300, 64), (2100, 260, 128), (2050, 129, 256), (5000, 2060, 50), (9001, 5, 40)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", SIZES)
def test_sizes_and_types(gsb, dt, N, V, D):
    x, w, t = make(N, V, D, dt, seed=N + V + D, ignored=0.1 if N > 4 else 0.0)
    check(gsb, x, w, t, scale=0.75)
    gsb.check_async_errors()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [40, 64, 128, 200, 272])
def test_long_sums_and_several_pieces(gsb, dt, D):
    """Every CTA runs over dozens of tiles (fp32 sums leave the accumulators several times), and the wide
    form takes the vocabulary in more than one piece."""
    x, w, t = make(5000, 8000, D, dt, seed=D, ignored=0.2)
    check(gsb, x, w, t)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(1, 5000, 128), (3, 129, 40), (200, 2500, 48), (300, 3001, 128), (257, 2100, 256), (140, 9000, 100),
                                   (70, 3000, 260), (300, 1000, 256), (400, 250, 90), (500, 47, 200), (500, 300, 60)])
def test_scores_without_gradients(gsb, dt, N, V, D):
    """No gradient is asked for: the pass that only keeps statistics, and with it dW alone."""
    x, w, t = make(N, V, D, dt, seed=V, ignored=0.1 if N > 4 else 0.0)
    t[0] = V - 1
    f = Formula(x, w, t, 0.9, dt)
    with torch.no_grad():
        within(gsb.ops.linear_cross_entropy(x, w.requires_grad_(), t, scale=0.9, reduction="none"), f.loss, f.loss_tol, "loss")
    (dw,) = torch.autograd.grad(gsb.ops.linear_cross_entropy(x, w, t, scale=0.9, reduction="sum"), [w])
    _, _, want, tol = f.grads(torch.ones(N, device="cuda"), dt)
    within(dw, want, tol, "dW")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V,scale", [(501, 1.0), (2200, 1.0), (501, -0.5), (2200, -0.5), (70, 0.0)])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions_upstream_gradients_and_signs(gsb, dt, reduction, V, scale):
    x, w, t = make(200, V, 96, dt, seed=5, ignored=0.3)
    up = torch.randn(200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) if reduction == "none" else -2.5
    check(gsb, x, w, t, scale=scale, reduction=reduction, up=up)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(300, 400, 64), (300, 400, 128), (300, 400, 300), (2100, 2100, 100), (200, 2100, 256)])
def test_rows_that_do_not_count_hide_what_they_hold(gsb, dt, N, V, D):
    x, w, t = make(N, V, D, dt, seed=6, ignored=0.5)
    clean = check(gsb, x, w, t)
    dirty = x.clone()
    dirty[t < 0] = float("nan")
    dirty[(t < 0).nonzero()[0, 0]] = float("inf")
    again = check(gsb, dirty, w, t)
    for a, b in zip(clean, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", DTYPES)
def test_no_row_counts(gsb, dt):
    x, w, _ = make(150, 300, 64, dt, seed=7)
    t = torch.full((150,), -1, device="cuda")
    for reduction in ("mean", "sum", "none"):
        loss, dx, dw = check(gsb, x, w, t, reduction=reduction)
        assert not bool(loss.any()) and not bool(dx.any()) and not bool(dw.any())


def test_no_rows_at_all(gsb):
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.randn(30, 64, device="cuda", requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    loss = gsb.ops.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert float(loss) == 0.0 and dx.shape == (0, 64) and not bool(dw.any())
    assert gsb.ops.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)


@pytest.mark.parametrize("dt", DTYPES)
def test_targets_outside_the_vocabulary_do_not_count_and_are_reported(gsb, dt):
    x, w, t = make(90, 200, 64, dt, seed=8)
    t[5], t[6] = 200, -7
    check(gsb, x, w, t)
    with pytest.raises(RuntimeError):
        gsb.check_async_errors()
    t[5], t[6] = -100, -100
    loss = gsb.ops.linear_cross_entropy(x, w, t, ignore_index=-100)
    assert bool(torch.isfinite(loss))
    gsb.check_async_errors()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V,D", [(2999, 64), (999, 64), (999, 128), (2999, 256), (47, 320)])
def test_far_apart_logits(gsb, dt, V, D):
    """One row's logits span hundreds and grow along the vocabulary, so that the running maximum moves in
    every piece; another row's all lie far below zero."""
    x = torch.zeros(4, D, device="cuda")
    w = torch.zeros(V, D, device="cuda")
    w[:, 0] = torch.linspace(0, 16, V, device="cuda")
    w[:, 1] = 1.0
    x[0, 0], x[1, 0], x[2, 1], x[3, 0] = 30.0, -30.0, -500.0, 0.01
    t = torch.tensor([V - 1, 0, 17, V // 2], device="cuda")
    check(gsb, x.to(dt), w.to(dt), t)


@pytest.mark.parametrize("dt", DTYPES)
def test_values_that_are_not_finite_reach_the_loss(gsb, dt):
    x, w, t = make(140, 300, 64, dt, seed=9)
    x[3, 5] = float("nan")
    w[299, 7] = float("inf")
    loss = gsb.ops.linear_cross_entropy(x, w, t, reduction="none")
    assert bool(torch.isnan(loss[3]))
    inf = x[:, 7] > 0
    assert not bool(torch.isfinite(loss[inf]).any())


@pytest.mark.parametrize("dt", DTYPES)
def test_views(gsb, dt):
    """Column slices, transposed tables, strided rows and leading dimensions give what their copies give."""
    x, w, t = make(96, 260, 72, dt, seed=10)

    def value(x, w, t):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = gsb.ops.linear_cross_entropy(x, w, t, reduction="none")
        return (loss.detach(),) + torch.autograd.grad(loss.sum(), [x, w])

    want = value(x, w, t)
    wide_x = torch.randn(96, 100, device="cuda").to(dt)
    wide_x[:, 13:85] = x
    wide_w = torch.randn(260, 75, device="cuda").to(dt)
    wide_w[:, 1:73] = w
    off = torch.empty(96 * 72 + 1, device="cuda", dtype=dt)[1:].view(96, 72).copy_(x)
    for xx, ww in ((wide_x[:, 13:85], w), (x, wide_w[:, 1:73]), (x.t().contiguous().t(), w), (off, w),
                   (x, w.t().contiguous().t()), (x.repeat_interleave(2, 0)[::2], w.repeat_interleave(3, 0)[::3])):
        for a, b in zip(value(xx, ww, t), want):
            assert torch.equal(a, b)
    got = value(x.view(8, 12, 72), w, t.view(8, 12))
    assert torch.equal(got[0], want[0].view(8, 12)) and torch.equal(got[1], want[1].view(8, 12, 72)) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("dt", DTYPES)
def test_one_of_the_gradients(gsb, dt):
    x, w, t = make(200, 300, 128, dt, seed=11)
    both = check(gsb, x, w, t)
    xl = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(gsb.ops.linear_cross_entropy(xl, w, t), [xl])
    wl = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(gsb.ops.linear_cross_entropy(x, wl, t), [wl])
    assert torch.equal(dx, both[1])
    # without a gradient for x the forward pass adds the log-sum-exp in another order, and dW is made
    # from it: each of the two lies within the tolerance of the formula, not at the same bits
    f = Formula(x, w, t, 1.0, dt)
    g = torch.full((200,), 1.0 / int(f.live.sum()), device="cuda")
    within(dw, f.grads(g, dt)[2], f.grads(g, dt)[3], "dW alone")
    tied = w[:200].clone().requires_grad_()     # one leaf on both sides: the gradients add up
    (d,) = torch.autograd.grad(gsb.ops.linear_cross_entropy(tied, tied, t % 200), [tied])
    a, b = tied.detach().clone().requires_grad_(), tied.detach().clone().requires_grad_()
    da, db = torch.autograd.grad(gsb.ops.linear_cross_entropy(a, b, t % 200), [a, b])
    assert torch.equal(d, da + db)


def test_gradient_against_differences(gsb):
    """Central differences of the 64-bit mean of the rows' losses: the third derivative along a unit
    coordinate is at most 2 (s w)^3, so a step h costs h^2 (s |w|max)^3 / 3; the losses carry loss_tol."""
    x, w, t = make(6, 50, 8, torch.float32, seed=12)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(gsb.ops.linear_cross_entropy(xl, wl, t, reduction="sum"), [xl, wl])
    h = 2.0 ** -5

    def total(a, b):
        return float(gsb.ops.linear_cross_entropy(a, b, t, reduction="none").double().sum())

    f = Formula(x, w, t, 1.0, torch.float32)
    noise = 2 * float(f.loss_tol.sum()) / (2 * h)
    for leaf, grad, other in ((x, dx, w), (w, dw, x)):
        for i, j in ((0, 0), (3, 5), (5, 7)):
            lo, hi = leaf.clone(), leaf.clone()
            lo[i, j] -= h
            hi[i, j] += h
            step = float((hi[i, j] - lo[i, j]).double())
            d = (total(hi, w) - total(lo, w)) / step if leaf is x else (total(x, hi) - total(x, lo)) / step
            bound = h * h * float(other.abs().max() + h) ** 3 / 3 * (1 if leaf is x else 6)
            assert abs(d - float(grad[i, j])) <= bound + noise


def test_streams_and_captured_graphs(gsb):
    x, w, t = make(300, 900, 128, torch.bfloat16, seed=13, ignored=0.1)
    want = check(gsb, x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = gsb.ops.linear_cross_entropy(xs, ws, t)
        got = (loss.detach(),) + torch.autograd.grad(loss, [xs, ws])
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss = gsb.ops.linear_cross_entropy(xs, ws, t)
            out = (loss.detach(),) + torch.autograd.grad(loss, [xs, ws])
        graphs.append((g, out))
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        for a, b in zip(want, out):
            assert torch.equal(a, b)


def test_refusals(gsb):
    x, w, t = make(4, 6, 8, torch.float32)
    for bad in (lambda: gsb.ops.linear_cross_entropy(x.double(), w.double(), t),
                lambda: gsb.ops.linear_cross_entropy(x.half(), w, t),
                lambda: gsb.ops.linear_cross_entropy(x, w[:, :7], t),
                lambda: gsb.ops.linear_cross_entropy(x, w[:0], t),
                lambda: gsb.ops.linear_cross_entropy(x, w.cpu(), t),
                lambda: gsb.ops.linear_cross_entropy(x, w, t.int()),
                lambda: gsb.ops.linear_cross_entropy(x, w, t, scale=math.inf)):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: gsb.ops.linear_cross_entropy(x, w, t[:3]),
                lambda: gsb.ops.linear_cross_entropy(x, w, t, reduction="max")):
        with pytest.raises(ValueError):
            bad()
