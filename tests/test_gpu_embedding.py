"""Embedding lookup and its gradient by sorted ids, against 64-bit sums on the host.

Tolerances.  The lookup multiplies in 32 bits and rounds once: one 32-bit rounding (2^-24) and one
of the type (half a step).  The gradient adds the c rows of an id in 32 bits: every term passes at
most c additions and one product, so its error is at most (c + 1) 2^-24 of the sum of magnitudes,
and the result is rounded once to the type.  fp16 results near zero are rounded to a multiple of
2^-24, by at most 2^-25."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def make(dt, rows, D, n, seed, hub=0.0, padding=0.0, bad=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(rows, D, generator=g).to(dt)
    idx = torch.randint(0, max(rows, 1), (n,), generator=g)
    if hub:
        idx[torch.rand(n, generator=g) < hub] = rows // 2
    if padding:
        idx[torch.rand(n, generator=g) < padding] = -1
    if bad:
        idx[torch.randint(0, n, (bad,), generator=g)] = rows + 3
    grad = torch.randn(n, D, generator=g).to(dt)
    return w, idx, grad


def expected(idx, grad, rows, scale):
    live = (idx >= 0) & (idx < rows)
    g = grad.double()[live] * scale
    want = torch.zeros(rows, grad.shape[-1], dtype=torch.float64).index_add_(0, idx[live], g)
    mag = torch.zeros_like(want).index_add_(0, idx[live], g.abs())
    count = torch.bincount(idx[live], minlength=rows).double()
    return want, mag, count


def check_grad(got, idx, grad, rows, scale, dt):
    want, mag, count = expected(idx, grad, rows, scale)
    tol = (count[:, None] + 1) * F32 * mag
    tol = tol + half_step(dt) * (want.abs() + tol) + (2.0 ** -25 if dt == torch.float16 else 0)
    assert got.dtype == dt
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,D,n,scale", [(1, 1, 1, 1.0), (7, 3, 40, 2.0), (1000, 100, 333, 0.5), (50, 64, 4096, 1.0),
                                            (300, 128, 4097, 8.0), (70001, 99, 20011, 1.0), (2000, 516, 3000, 0.3),
                                            (300000, 8, 100003, 1.0)])
def test_lookup_and_dense_gradient(gsb, dt, rows, D, n, scale):
    w, idx, grad = make(dt, rows, D, n, seed=rows + D, hub=0.2, padding=0.05)
    wd = w.cuda().requires_grad_()
    out = gsb.ops.embedding(wd, idx.cuda(), scale=scale)
    want = w.double()[idx.clamp(min=0)] * scale * (idx >= 0).double()[:, None]
    tol = (half_step(dt) + (0 if scale == 1 else 1.01 * F32)) * want.abs() + (2.0 ** -25 if dt == torch.float16 else 0)
    assert bool(((out.detach().cpu().double() - want).abs() <= tol).all())
    if scale == 1.0:
        assert torch.equal(out.detach().cpu(), torch.where((idx >= 0)[:, None], w[idx.clamp(min=0)], torch.zeros((), dtype=dt)))
    (dw,) = torch.autograd.grad(out, [wd], grad.cuda())
    check_grad(dw, idx, grad, rows, scale, dt)
    gsb.check_async_errors()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,D,n", [(5, 4, 1), (1000, 100, 4096), (1 << 17, 7, 30011), (90, 64, 200003)])
def test_sparse_gradient(gsb, dt, rows, D, n):
    w, idx, grad = make(dt, rows, D, n, seed=n, hub=0.3, padding=0.1 if n > 1 else 0.0)
    wd = w.cuda().requires_grad_()
    out = gsb.ops.embedding(wd, idx.cuda(), scale=0.5, sparse=True)
    (dw,) = torch.autograd.grad(out, [wd], grad.cuda())
    assert dw.is_sparse and dw.is_coalesced() and dw.shape == (rows, D)
    ids = dw.indices()[0].cpu()
    assert torch.equal(ids, torch.unique(idx[idx >= 0]))
    check_grad(dw.to_dense(), idx, grad, rows, 0.5, dt)
    dense = gsb.ops.embedding(wd, idx.cuda(), scale=0.5)
    (dd,) = torch.autograd.grad(dense, [wd], grad.cuda())
    assert torch.equal(dd[ids.cuda()], dw.values())


@pytest.mark.parametrize("n,hub", [(100000, 1.0), (300000, 0.5), (70000, 0.999)])
def test_hub_rows_are_summed_in_a_fixed_order(gsb, n, hub):
    """An id that fills the batch passes every level of partial sums; twice the same bits."""
    w, idx, grad = make(torch.float32, 1000, 33, n, seed=4, hub=hub)
    a, b = (torch.ops.gs_ops._CAPI_EmbeddingGrad(grad.cuda(), idx.cuda(), 1000, 1.0, -1) for _ in range(2))
    assert torch.equal(a, b)
    check_grad(a, idx, grad, 1000, 1.0, torch.float32)


def test_all_ids_are_padding_or_none(gsb):
    w = torch.randn(10, 6, device="cuda", requires_grad=True)
    for idx in (torch.full((5000,), -1, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")):
        for sparse in (False, True):
            out = gsb.ops.embedding(w, idx, sparse=sparse)
            assert out.shape == (idx.numel(), 6) and not bool(out.any())
            (dw,) = torch.autograd.grad(out, [w], torch.full_like(out, float("nan")))
            assert not bool(dw.to_dense().any()), "padding rows have no gradient, not even a NaN one"
    gsb.check_async_errors()
    out = gsb.ops.embedding(w, torch.tensor([3, 4, 3], device="cuda"), padding_idx=3)
    assert not bool(out[0].any()) and torch.equal(out[1], w[4])


def test_bad_ids_are_zero_rows_and_reported(gsb):
    w, idx, grad = make(torch.float32, 40, 12, 300, seed=9, bad=5)
    wd = w.cuda().requires_grad_()
    out = gsb.ops.embedding(wd, idx.cuda())
    assert not bool(out[(idx >= 40).cuda()].any())
    with pytest.raises(RuntimeError):
        gsb.check_async_errors()
    (dw,) = torch.autograd.grad(out, [wd], grad.cuda())
    with pytest.raises(RuntimeError):
        gsb.check_async_errors()
    check_grad(dw, idx, grad, 40, 1.0, torch.float32)


def test_shapes_strides_and_offsets(gsb):
    """Ids of any shape and order, a table that is a column slice, a row slice or transposed, and a
    gradient that is a broadcast scalar."""
    big = torch.randn(50, 40, device="cuda")
    idx = torch.randint(0, 50, (6, 9), device="cuda").t()
    for w in (big[:, 3:16], big[:, 8:24], big[5:, :], big[::2], torch.randn(13, 50, device="cuda").t()):
        ids = idx % w.shape[0]
        out = gsb.ops.embedding(w, ids)
        assert out.shape == (9, 6, w.shape[1]) and torch.equal(out, w[ids])
    w = big.clone().requires_grad_()
    gsb.ops.embedding(w, idx).sum().backward()
    count = torch.bincount(idx.reshape(-1), minlength=50).float()
    assert torch.equal(w.grad, count[:, None].expand(50, 40))
    base = torch.randn(50 * 8 + 1, device="cuda")
    w = base[1:].view(50, 8)           # rows that start 4 bytes off a 16-byte boundary
    assert torch.equal(gsb.ops.embedding(w, idx), w[idx])


def test_gradient_against_differences(gsb):
    """The loss is linear in the table, so a difference of any width is exact up to rounding: for a
    step h the two losses differ by h * dw, each with at most 40 products and additions in 32 bits."""
    w, idx, grad = make(torch.float32, 6, 5, 8, seed=2)
    gd = grad.cuda()
    wd = w.cuda().requires_grad_()
    (dw,) = torch.autograd.grad(gsb.ops.embedding(wd, idx.cuda(), scale=1.5), [wd], gd)
    for v, c in ((0, 0), (3, 2), (5, 4)):
        h = 2.0
        lo, hi = w.clone(), w.clone()
        lo[v, c] -= h
        hi[v, c] += h
        f = [(gsb.ops.embedding(t.cuda(), idx.cuda(), scale=1.5).double() * gd.double()).sum() for t in (lo, hi)]
        size = 1.5 * (w.abs().max() + h) * grad.abs().sum()
        assert abs(float(f[1] - f[0]) / (2 * h) - float(dw[v, c])) <= 40 * F32 * float(size)


def test_streams_and_captured_graphs(gsb):
    """Forward and backward on a side stream and replayed from a CUDA graph while an eager graph of the
    same table lives: the same bits."""
    w, idx, grad = make(torch.bfloat16, 5000, 64, 9001, seed=12, hub=0.1)
    wd, ix, gd = w.cuda().requires_grad_(), idx.cuda(), grad.cuda()
    eager = gsb.ops.embedding(wd, ix)
    (want,) = torch.autograd.grad(eager, [wd], gd, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        (dw,) = torch.autograd.grad(gsb.ops.embedding(wd, ix), [wd], gd)
    side.synchronize()
    assert torch.equal(dw, want)
    leaf = wd.detach().clone().requires_grad_()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = gsb.ops.embedding(leaf, ix)
            (dw,) = torch.autograd.grad(out, [leaf], gd)
        graphs.append((g, out, dw))
    for _ in range(2):
        for g, out, dw in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out, dw in graphs:
            assert torch.equal(out, eager) and torch.equal(dw, want)


def test_refusals(gsb):
    w = torch.randn(4, 4, device="cuda")
    i = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: gsb.ops.embedding(w.double(), i), lambda: gsb.ops.embedding(w, i.int()),
                lambda: gsb.ops.embedding(w.cpu(), i), lambda: gsb.ops.embedding(w, i.cpu()),
                lambda: gsb.ops.embedding(w.view(2, 2, 4), i), lambda: gsb.ops.embedding(w, i, scale=float("nan")),
                lambda: torch.ops.gs_ops._CAPI_EmbeddingGrad(w, i, 4, 1.0, -1)):
        with pytest.raises(RuntimeError):
            bad()
