"""Dropout from the counter-based streams against the oracle's Philox: the mask has to be the one the
definition names, element for element; the kept values are one 32-bit product rounded once."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def numbers(oracle, n, seed, stream):
    out = np.empty((n + 7) // 8 * 8, dtype=np.int64)
    key = (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)
    for g in range((n + 7) // 8):
        w = np.asarray(oracle.philox4x32_10((g & 0xFFFFFFFF, g >> 32, 0, stream & 0xFFFFFFFF), key), dtype=np.int64)
        out[8 * g:8 * g + 8:2] = w & 0xFFFF
        out[8 * g + 1:8 * g + 8:2] = w >> 16
    return out[:n]


def want(oracle, x, p, seed, stream):
    t = int(np.floor(p * 65536 + 0.5))
    keep = torch.from_numpy(numbers(oracle, x.numel(), seed, stream) >= t).view(x.shape)
    mul = 65536.0 / (65536 - t) if t < 65536 else 0.0
    return keep, torch.where(keep, x.double() * mul, torch.zeros((), dtype=torch.float64))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((7,), 0.25), ((8,), 0.9), ((33, 9), 0.1), ((500, 100), 0.5),
                                     ((3, 5, 77), 1e-3), ((64, 64), 1.0)])
def test_mask_and_values_both_directions(gsb, oracle, dt, shape, p):
    g = torch.Generator().manual_seed(3)
    x, dy = torch.randn(shape, generator=g).to(dt), torch.randn(shape, generator=g).to(dt)
    xd = x.cuda().requires_grad_()
    seed, stream = 0x1234567890AB, 42
    y = gsb.ops.dropout(xd, p, seed=seed, stream=stream)
    (dx,) = torch.autograd.grad(y, [xd], dy.cuda())
    # the factor and the product are rounded to 32 bits, the result to the type
    rel = torch.finfo(dt).eps / 2 + 2.01 * 2.0 ** -24
    for got, src in ((y, x), (dx, dy)):
        keep, ref = want(oracle, src, p, seed, stream)
        got = got.detach().cpu()
        assert got.dtype == dt and got.shape == src.shape
        assert not bool(got[~keep].any())
        assert bool(((got.double() - ref).abs() <= rel * ref.abs() + (2.0 ** -25 if dt == torch.float16 else 0)).all())


def test_dropped_places_hide_infinities_and_nan(gsb, oracle):
    x = torch.full((4000,), float("nan"))
    x[::2] = float("inf")
    keep, _ = want(oracle, torch.zeros(4000), 0.5, 5, 6)
    y = gsb.ops.dropout(x.cuda(), 0.5, seed=5, stream=6).cpu()
    assert bool((y[~keep] == 0).all()) and not bool(torch.isfinite(y[keep]).any())


def test_share_of_dropped_elements(gsb):
    """n = 2^22 independent elements: the count is binomial, six standard deviations allowed."""
    n = 1 << 22
    for p in (0.1, 0.5, 0.9):
        y = gsb.ops.dropout(torch.ones(n, device="cuda"), p, seed=1, stream=0)
        t = int(p * 65536 + 0.5) / 65536
        assert abs(int((y == 0).sum()) - n * t) <= 6 * (n * t * (1 - t)) ** 0.5


def test_default_state_advances_and_repeats(gsb):
    x = torch.ones(1000, device="cuda")
    torch.ops.gs_ops._CAPI_SetDropoutSeed(99)
    a, b = gsb.ops.dropout(x), gsb.ops.dropout(x)
    torch.ops.gs_ops._CAPI_SetDropoutSeed(99)
    c = gsb.ops.dropout(x)
    assert torch.equal(a, c) and not torch.equal(a, b)
    assert torch.equal(a, gsb.ops.dropout(x, seed=99, stream=0))
    assert gsb.ops.dropout(x, training=False) is x and gsb.ops.dropout(x, 0.0) is x


def test_views_and_unaligned_storage(gsb, oracle):
    base = torch.randn(1001, device="cuda").half()
    for x in (base[1:], base[1:1000].view(333, 3).t(), base[:1000:3], base[:0]):
        y = gsb.ops.dropout(x, 0.3, seed=8, stream=1)
        _, ref = want(oracle, x.cpu().contiguous(), 0.3, 8, 1)
        assert y.shape == x.shape
        assert bool(((y.cpu().double() - ref).abs() <= (2.0 ** -11 + 2.01 * 2.0 ** -24) * ref.abs() + 2.0 ** -25).all())


def test_step_gives_every_replay_its_own_mask(gsb):
    x = torch.ones(4096, device="cuda", requires_grad=True)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = gsb.ops.dropout(x, 0.5, seed=3, stream=10, step=step)
        (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
        step.add_(1)
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        want_k = gsb.ops.dropout(x.detach(), 0.5, seed=3, stream=10 + k)
        assert torch.equal(y, want_k) and torch.equal(dx, want_k)
    # a step changed between the passes would draw another mask: autograd refuses
    y = gsb.ops.dropout(x, 0.5, seed=3, stream=10, step=step)
    step.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_refusals(gsb):
    x = torch.ones(4, device="cuda")
    for bad in (lambda: gsb.ops.dropout(x, 1.5), lambda: gsb.ops.dropout(x, -0.1), lambda: gsb.ops.dropout(x, seed=1),
                lambda: gsb.ops.dropout(x, float("nan"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: gsb.ops.dropout(x.double(), 0.5), lambda: gsb.ops.dropout(x.cpu(), 0.5),
                lambda: gsb.ops.dropout(x, 0.5, step=torch.zeros(2, dtype=torch.int64, device="cuda"), seed=1, stream=1)):
        with pytest.raises(RuntimeError):
            bad()
