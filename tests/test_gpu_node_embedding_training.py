"""The operators on learned node values together, as a walk-trained embedding uses them: node2vec walks
from the library, pairs of a node and the next, their vectors looked up, dropped out and scored against
every node.  One step's gradients against the formula in 64 bits, and the step recorded into a CUDA graph."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -23


@pytest.fixture(scope="module")
def pairs(gsb):
    rng = np.random.default_rng(3)
    n = 700
    deg = rng.integers(1, 12, n)
    indptr = np.concatenate([[0], np.cumsum(deg)]).astype(np.int64)
    indices = rng.integers(0, n, indptr[-1]).astype(np.int64)
    deg0 = indptr[1:] - indptr[:-1]
    assert deg0.min() >= 1
    m = gsb.Matrix()
    m.load_graph("CSC", [torch.as_tensor(indptr).cuda(), torch.as_tensor(indices).cuda()])
    m._graph._CAPI_SortCSCIndices()
    m._graph._CAPI_SetSeed(5)
    walks = m.random_walk(torch.arange(0, n, 3, device="cuda"), 6).reshape(7, -1)
    centre, context = walks[:-1].reshape(-1).contiguous(), walks[1:].reshape(-1).contiguous()
    context = torch.where(centre < 0, torch.full_like(context, -1), context)
    return n, centre, context


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sparse", [False, True])
def test_one_step_against_the_formula(gsb, pairs, dt, sparse):
    n, centre, context = pairs
    D, p, scale = 64, 0.25, 0.5
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randn(n, D, device="cuda", generator=g).to(dt).requires_grad_()
    out = (torch.randn(n, D, device="cuda", generator=g) * D ** -0.5).to(dt).requires_grad_()
    h = gsb.ops.embedding(table, centre, scale=2.0, sparse=sparse)
    x = gsb.ops.dropout(h, p, seed=9, stream=4)
    loss = gsb.ops.linear_cross_entropy(x, out, context, scale=scale)
    d_table, d_out = torch.autograd.grad(loss, [table, out])
    gsb.check_async_errors()
    # the formula, from the values the operators pass on (each is rounded to the type once)
    live = context >= 0
    mask = (gsb.ops.dropout(torch.ones_like(h), p, seed=9, stream=4) != 0).double() * (65536.0 / (65536 - 16384))
    H = (2.0 * table.detach().double()[centre.clamp(min=0)] * (centre >= 0).double()[:, None])
    X = H * mask
    W = out.detach().double()
    l = scale * X @ W.T
    lse = torch.logsumexp(l, 1)
    count = int(live.sum())
    pr = torch.exp(l - lse[:, None])
    hot = torch.zeros_like(pr)
    hot[torch.arange(len(centre), device="cuda"), context.clamp(min=0)] = 1.0
    gl = live.double() / count * scale
    cell = (pr - hot) * gl[:, None]
    want_out = cell.T @ X
    dX = cell @ W
    dH = dX * mask * 2.0
    want_table = torch.zeros(n, D, dtype=torch.float64, device="cuda").index_add_(0, centre.clamp(min=0), dH * (centre >= 0).double()[:, None])
    # A chain of roundings, h half a step of the type: the lookup and the dropout are off by h each (fp32
    # products u each), so a logit by e = (2 h + (D + 4) u) times the sum of its magnitudes, p by
    # (2 e + 8 u) relative, and every value that is passed on by another h.
    h_ = torch.finfo(dt).eps / 2
    e = ((2 * h_ + (D + 4) * U) * scale * X.abs() @ W.abs().T).amax(1, keepdim=True)
    rel = 2 * e + 8 * U + 3 * h_ + n * U
    mag = (pr * rel + hot * (2 * h_ + 4 * U)) * gl[:, None]
    tiny = 2.0 ** -24 if dt == torch.float16 else 0.0
    tol_out = mag.T @ X.abs() + (cell.abs().T @ X.abs()) * 2 * h_ + (len(centre) * U + h_) * (cell.abs().T @ X.abs()) + tiny
    tol_dX = mag @ W.abs() + h_ * dX.abs() + tiny
    tol_dH = (tol_dX + (h_ + 2 * U) * dX.abs()) * mask * 2.0 + 2 * tiny
    many = torch.bincount(centre.clamp(min=0), minlength=n).double()[:, None]
    size = torch.zeros_like(want_table).index_add_(0, centre.clamp(min=0), dH.abs())
    tol_table = torch.zeros_like(want_table).index_add_(0, centre.clamp(min=0), tol_dH) + (many + 1) * U * size + h_ * want_table.abs() + tiny
    tol_loss = float((2 * e + 8 * U).max()) + U * n
    assert abs(float(loss.detach().double()) - float(((lse - (l * hot).sum(1)) * live).sum() / count)) <= tol_loss
    d_table = d_table.to_dense() if sparse else d_table
    for got, want, tol, what in ((d_out, want_out, tol_out, "output table"), (d_table, want_table, tol_table, "input table")):
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), "%s: %g over" % (what, float((err - tol).max()))


def test_a_recorded_step_replays_with_new_masks(gsb, pairs):
    n, centre, context = pairs
    table = torch.randn(n, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = torch.randn(n, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def run(stream, step=None):
        x = gsb.ops.dropout(gsb.ops.embedding(table, centre), 0.5, seed=2, stream=stream, step=step)
        loss = gsb.ops.linear_cross_entropy(x, out, context)
        return (loss.detach(),) + torch.autograd.grad(loss, [table, out])

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run(100, step)
        step.add_(1)
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, run(100 + k)):
            assert torch.equal(a, b)


def test_every_operator_on_two_streams_at_once(gsb, pairs):
    n, centre, context = pairs
    tables = [torch.randn(n, 96, device="cuda").half().requires_grad_() for _ in range(2)]
    outs = [torch.randn(n, 96, device="cuda").half().requires_grad_() for _ in range(2)]

    def run(i):
        x = gsb.ops.dropout(gsb.ops.embedding(tables[i], centre), 0.1, seed=1, stream=i)
        loss = gsb.ops.linear_cross_entropy(x, outs[i], context, scale=0.1)
        return (loss.detach(),) + torch.autograd.grad(loss, [tables[i], outs[i]])

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)
