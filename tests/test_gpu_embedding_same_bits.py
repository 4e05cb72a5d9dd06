"""The order of the embedding gradient's sums depends on the ids and the sizes, not on where the gradient lies in
memory: a view that begins inside a buffer gives the bits of its copy, also for ids that fill the batch."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [1, 8, 24, 40, 64, 100, 256, 520])
@pytest.mark.parametrize("n,hub", [(60000, 0.999), (200000, 0.6), (3000, 1.0)])
def test_a_gradient_off_a_boundary(gsb, dt, D, n, hub):
    g = torch.Generator(device="cuda").manual_seed(D + n)
    idx = torch.randint(0, 500, (n,), device="cuda", generator=g)
    idx[torch.rand(n, device="cuda", generator=g) < hub] = 77
    grad = torch.randn(n, D, device="cuda", generator=g).to(dt)
    want = torch.ops.gs_ops._CAPI_EmbeddingGrad(grad, idx, 500, 0.5, -1)
    for off in (1, 2, 4):
        moved = torch.empty(n * D + off, dtype=dt, device="cuda")[off:].view(n, D).copy_(grad)
        assert torch.equal(torch.ops.gs_ops._CAPI_EmbeddingGrad(moved, idx, 500, 0.5, -1), want)
        ids, rows = torch.ops.gs_ops._CAPI_EmbeddingSparseGrad(moved, idx, 500, 0.5, -1)
        assert torch.equal(rows, want[ids])
