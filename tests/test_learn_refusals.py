"""Argument checks of the operators on learned node values that need no GPU."""
import ctypes as C

import pytest
import torch

from tests import abi


def test_c_entry_points_check_their_arguments():
    L = abi.lib()
    f, d, nul = C.c_float(1.0), C.c_double(0.5), None
    ok, invalid = 0, 1
    assert L.gsb_embedding(nul, 0, abi.i64(4), abi.i64(2), abi.i64(4), nul, abi.i64(0), f, abi.i64(-1), nul, nul, nul) == ok
    assert L.gsb_embedding(nul, 0, abi.i64(4), abi.i64(2), abi.i64(4), nul, abi.i64(3), f, abi.i64(-1), nul, nul, nul) == invalid
    assert L.gsb_embedding(nul, 0, abi.i64(3), abi.i64(2), abi.i64(4), nul, abi.i64(0), f, abi.i64(-1), nul, nul, nul) == invalid
    assert L.gsb_embedding_grad(nul, 7, abi.i64(4), nul, abi.i64(0), abi.i64(0), f, abi.i64(-1), nul, nul, C.c_size_t(0),
                                nul, nul) == invalid
    assert L.gsb_embedding_grad_workspace_bytes(abi.i64(1 << 31), abi.i64(10), abi.i64(4)) == 0
    assert L.gsb_embedding_grad_workspace_bytes(abi.i64(1000), abi.i64(10), abi.i64(4)) > 0
    assert L.gsb_dropout(nul, 0, abi.i64(0), d, C.c_uint64(1), C.c_uint32(1), nul, nul, nul) == ok
    assert L.gsb_dropout(nul, 0, abi.i64(4), d, C.c_uint64(1), C.c_uint32(1), nul, nul, nul) == invalid
    for p in (-0.1, 1.1, float("nan")):
        assert L.gsb_dropout(nul, 0, abi.i64(0), C.c_double(p), C.c_uint64(1), C.c_uint32(1), nul, nul, nul) == invalid
    lce = lambda x, dt, N, V, D: L.gsb_linear_ce(x, dt, abi.i64(D), abi.i64(N), x, abi.i64(D), abi.i64(V), abi.i64(D), nul,
                                                 abi.i64(-1), f, nul, nul, nul, nul, C.c_size_t(0), nul, nul)
    assert lce(nul, 0, 0, 5, 4) == ok
    assert lce(nul, 0, 3, 5, 4) == invalid and lce(nul, 9, 0, 5, 4) == invalid
    assert lce(nul, 0, 0, 0, 4) == invalid and lce(nul, 0, 0, 5, 0) == invalid
    assert L.gsb_linear_ce_workspace_bytes(0, nul, abi.i64(4), abi.i64(1 << 31), abi.i64(5), abi.i64(4), 0) == 0
    for n in (0, 1):
        for dt in (0, 1, 2):
            L.gsb_linear_ce_workspace_bytes(dt, nul, abi.i64(4), abi.i64(n), abi.i64(5), abi.i64(4), 1)
            L.gsb_linear_ce_grad_workspace_bytes(dt, nul, abi.i64(4), abi.i64(n), abi.i64(5), abi.i64(4), 1, 1, 1)
        L.gsb_embedding_grad_workspace_bytes(abi.i64(n), abi.i64(0), abi.i64(0))
    assert L.gsb_linear_ce_workspace_bytes(0, nul, abi.i64(4), abi.i64(100), abi.i64(5), abi.i64(4), 0) > 0


def test_there_is_no_cpu_path():
    import gsampler_b200 as gs

    w, i = torch.randn(4, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        gs.ops.embedding(w, i)
    with pytest.raises(RuntimeError):
        gs.ops.dropout(w, 0.5)
    with pytest.raises(RuntimeError):
        gs.ops.linear_cross_entropy(w, w, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        gs.ops.linear_cross_entropy(w, w, i)
    for p in (-0.5, 2.0, float("nan")):
        with pytest.raises(ValueError):
            gs.ops.dropout(w, p)
    with pytest.raises(ValueError):
        gs.ops.dropout(w, 0.5, stream=3)
