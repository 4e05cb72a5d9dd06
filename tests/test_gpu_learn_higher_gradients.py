"""Gradients of gradients and forward-mode tangents through the operators on learned node values: right, or
refused, and never dropped.  The lookup and dropout are linear, so their second gradients are the first ones of
the same maps: compared with torch's indexing and product on the same mask, in 64 bits.  Tolerance: the terms
pass at most 40 products and additions of 2^-24 each."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


def near(got, want, size):
    assert bool(((got.double() - want).abs() <= 40 * F32 * size).all())


def test_second_gradient_of_a_lookup_and_dropout(gsb):
    g = torch.Generator(device="cuda").manual_seed(4)
    table = torch.randn(20, 8, device="cuda", generator=g)
    idx = torch.randint(-1, 20, (12,), device="cuda", generator=g)
    v = torch.randn(20, 8, device="cuda", generator=g)
    mask = gsb.ops.dropout(torch.ones(12, 8, device="cuda"), 0.25, seed=3, stream=7)

    def second(t, lookup, drop):
        t = t.clone().requires_grad_()
        y = drop(lookup(t))
        (d,) = torch.autograd.grad((y ** 3).sum(), [t], create_graph=True)
        assert d.requires_grad
        (dd,) = torch.autograd.grad((d * v.to(d.dtype)).sum() + (d ** 2).sum(), [t], create_graph=True)
        (ddd,) = torch.autograd.grad(dd.sum(), [t])
        return d.detach(), dd.detach(), ddd

    got = second(table, lambda t: gsb.ops.embedding(t, idx, scale=1.5), lambda x: gsb.ops.dropout(x, 0.25, seed=3, stream=7))
    live = (idx >= 0).double()[:, None]
    want = second(table.double(), lambda t: 1.5 * t[idx.clamp(min=0)] * live, lambda x: x * mask.double())
    v.abs_()
    size = second(table.double().abs(), lambda t: 1.5 * t[idx.clamp(min=0)] * live, lambda x: x * mask.double())
    for a, b, c in zip(got, want, size):
        near(a, b, c)


def test_second_gradient_of_dropout_with_a_step(gsb):
    x = torch.randn(100, device="cuda", requires_grad=True)
    step = torch.full((1,), 5, dtype=torch.int64, device="cuda")
    (d,) = torch.autograd.grad((gsb.ops.dropout(x, 0.5, seed=1, stream=2, step=step) ** 2).sum(), [x], create_graph=True)
    (dd,) = torch.autograd.grad(d.sum(), [x])
    keep = gsb.ops.dropout(torch.ones(100, device="cuda"), 0.5, seed=1, stream=7)
    near(dd, 2 * keep.double() ** 2, 2 * keep.double() ** 2)


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("V,D", [(30, 16), (2100, 16), (30, 300)])
def test_the_losss_gradient_refuses_to_be_differentiated(gsb, reduction, V, D):
    x = torch.randn(10, D, device="cuda", requires_grad=True)
    w = torch.randn(V, D, device="cuda", requires_grad=True)
    t = torch.randint(0, V, (10,), device="cuda")
    loss = gsb.ops.linear_cross_entropy(x, w, t, reduction=reduction).sum()
    plain = torch.autograd.grad(loss, [x, w], retain_graph=True)
    graphed = torch.autograd.grad(loss, [x, w], create_graph=True)
    for a, b in zip(plain, graphed):
        assert torch.equal(a, b.detach()) and b.requires_grad
        with pytest.raises(RuntimeError, match="gradients of gradients"):
            torch.autograd.grad(b.square().sum(), [x])
    total = loss + graphed[0].square().sum()       # a penalty on the gradient
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        total.backward()


def test_the_sparse_gradient_refuses_to_be_differentiated(gsb):
    w = torch.randn(20, 4, device="cuda", requires_grad=True)
    idx = torch.tensor([3, 5, 3], device="cuda")
    out = gsb.ops.embedding(w, idx, sparse=True)
    (d,) = torch.autograd.grad((out ** 2).sum(), [w], create_graph=True)
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(d.to_dense().sum(), [w])
    out = gsb.ops.embedding(w, idx, sparse=True)   # linear use: nothing to differentiate, and no error
    (d,) = torch.autograd.grad(out.sum(), [w], create_graph=True)
    assert float(d.to_dense().sum()) == 12.0


def test_tangents_are_refused(gsb):
    w = torch.randn(20, 4, device="cuda")
    idx = torch.tensor([3, 5, 3], device="cuda")
    t = torch.tensor([0, 1, 2], device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: gsb.ops.embedding(dual, idx), lambda: gsb.ops.dropout(dual, 0.5),
                     lambda: gsb.ops.linear_cross_entropy(dual[:3], w, t), lambda: gsb.ops.linear_cross_entropy(w[:3], dual, t)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: gsb.ops.embedding(a, idx), (w,), (torch.ones_like(w),))
