"""dx of rows whose target is already likely: dx_i = g_i s (sum_{j != t} p_ij w_j - (1 - p_t) w_t), where both
parts are of the size of 1 - p_t, so an error of half a step of p_t is many times the gradient.

The values are small multiples of a power of two with few non-zeros, so that every product and every sum
of a logit is exact in 32 bits in any order.  What is left of the errors (u = 2^-23, h half a step of the type):
  logit   a_ij = 4 u |l_ij|          the factor to base 2 and its product
  lse     b_i  = u (V / 16 + 64) + 8 u max_j |l_ij|     sums in runs of 16 or more, exp, log, its 32 bits
  p_ij    relative r_ij = a_ij + b_i + 8 u, and h where the matrix units take it in 16 bits (q = 2^-31 for fp16)
  1 - p_t p_t r_it, and half a step of itself
  dx_i    |g_i s| (sum_{j != t} (p_ij (r_ij + h + V u) + q) |w_jd| + ((1 - p_t) h + p_t r_it + 4 u (1 - p_t)) |w_td|),
          then half a step of the type
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def table(V, D, seed):
    """Rows of 64 values n / 8, |n| <= 4 (all of D where D is smaller), zeros elsewhere."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randint(-4, 5, (V, D), device="cuda", generator=g).double() / 8
    if D > 64:
        w *= torch.rand(V, D, device="cuda", generator=g).argsort(1) < 64
    return w


def rows_with(w, targets, miss):
    """x_i = k w_t / 16 with the k for which 1 - p_t comes nearest to miss[i]."""
    k = torch.arange(4, 64, device="cuda").double() / 16
    x = torch.empty(len(targets), w.shape[1], dtype=torch.float64, device="cuda")
    for i, t in enumerate(targets.tolist()):
        l = k[:, None] * (w @ w[t])[None, :]
        others = l.clone()
        others[:, t] = -float("inf")
        m = torch.sigmoid(torch.logsumexp(others, 1) - l[:, t])
        x[i] = w[t] * k[(m.log() - torch.tensor(miss[i]).log()).abs().argmin()]
    return x


def expected(x, w, t, scale, g, dt):
    V = w.shape[0]
    l = scale * x @ w.T
    rows = torch.arange(len(t), device="cuda")
    lt = l[rows, t]
    lse = torch.logsumexp(l, 1)
    others = l.clone()
    others[rows, t] = -float("inf")
    p = torch.exp(others - lse[:, None])                            # zero at the target
    miss = torch.sigmoid(torch.logsumexp(others, 1) - lt)          # 1 - p_t, without cancellation
    b = U * (V / 16 + 64 + 8 * l.abs().amax(1))
    r = 4 * U * l.abs() + b[:, None] + 8 * U
    rt = 4 * U * lt.abs() + b + 8 * U
    h = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    q = 2.0 ** -31 if dt == torch.float16 else 0.0
    gs = (g.double() * scale)[:, None]
    dx = gs * (p @ w - miss[:, None] * w[t])
    tol = gs.abs() * ((p * (r + h + V * U) + q) @ w.abs() + (miss * (h + 4 * U) + (1 - miss) * rt)[:, None] * w[t].abs())
    tol = tol + torch.finfo(dt).eps / 2 * (dx.abs() + tol) + (2.0 ** -25 if dt == torch.float16 else 0)
    return dx, tol, miss


MISSES = [0.5, 0.1, 0.03, 0.01, 3e-3, 1e-3, 3e-4, 1e-4]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V,D,repeat", [(47, 64, 1), (47, 256, 40), (300, 128, 1), (1999, 64, 25), (2048, 100, 1),
                                        (2049, 64, 1), (3000, 128, 20), (2500, 256, 1), (700, 300, 10), (2600, 300, 1)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_rows_whose_target_is_likely(gsb, dt, V, D, repeat, reduction):
    w = table(V, D, V + D)
    miss = MISSES * (4 * repeat)
    gen = torch.Generator().manual_seed(V)
    t = torch.randint(0, V, (len(MISSES) * 4,), generator=gen).cuda()
    x = rows_with(w, t, miss[:len(t)]).repeat(repeat, 1)
    t = t.repeat(repeat)
    xl, wl = x.to(dt).requires_grad_(), w.to(dt).requires_grad_()
    assert torch.equal(xl.detach().double(), x) and torch.equal(wl.detach().double(), w), "the type holds the values"
    # fp16 holds gradients above 2^-14 with all its digits: the mean's are scaled as a training step scales them
    up = torch.ones(len(t), device="cuda") * 64 if reduction == "none" else torch.tensor(64.0 * len(t), device="cuda")
    g = torch.full((len(t),), 64.0, device="cuda")
    (dx,) = torch.autograd.grad(gsb.ops.linear_cross_entropy(xl, wl, t, reduction=reduction), [xl], up, retain_graph=True)
    want, tol, got_miss = expected(x, w, t, 1.0, g, dt)
    assert float(got_miss.min()) < 2e-4 and float(got_miss.max()) > 0.2, "the rows cover the range"
    err = (dx.double() - want).abs()
    worst = ((err - tol).amax(1) > 0).nonzero().flatten()
    assert worst.numel() == 0, "1 - p_t = %s: error %s of %s" % (
        got_miss[worst[:5]].tolist(), err[worst[:5]].amax(1).tolist(), want[worst[:5]].abs().amax(1).tolist())
    gsb.check_async_errors()
