"""A scale that is not finite, also after it became a float32, is refused by the C entries and before any of
them is reached."""
import ctypes as C

import pytest
import torch

from tests import abi

BAD = [float("inf"), -float("inf"), float("nan")]


@pytest.mark.parametrize("scale", BAD)
def test_c_entries_refuse_it(scale):
    L, f, nul, none = abi.lib(), C.c_float(scale), None, abi.i64(-1)
    four, zero = abi.i64(4), abi.i64(0)
    for dt in (0, 1, 2):
        assert L.gsb_embedding(nul, dt, four, four, four, nul, zero, f, none, nul, nul, nul) == 1
        assert L.gsb_embedding_grad(nul, dt, four, nul, zero, zero, f, none, nul, nul, C.c_size_t(0), nul, nul) == 1
        assert L.gsb_embedding_grad_rows(nul, dt, four, four, four, zero, f, nul, nul, C.c_size_t(0), nul) == 1
        assert L.gsb_linear_ce(nul, dt, four, zero, nul, four, four, four, nul, none, f, nul, nul, nul, nul, C.c_size_t(0), nul, nul) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("scale", BAD + [1e39, -1e300])
def test_operators_refuse_it(gsb, scale):
    w = torch.randn(4, 4, device="cuda")
    i = torch.zeros(3, dtype=torch.int64, device="cuda")
    for call in (lambda: gsb.ops.embedding(w, i, scale=scale), lambda: torch.ops.gs_ops._CAPI_EmbeddingGrad(w[:3], i, 4, scale, -1),
                 lambda: torch.ops.gs_ops._CAPI_EmbeddingSparseGrad(w[:3], i, 4, scale, -1),
                 lambda: gsb.ops.linear_cross_entropy(w[:3], w, i, scale=scale)):
        with pytest.raises(RuntimeError, match="scale must be finite"):
            call()
