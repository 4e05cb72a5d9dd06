"""The gradient entry that takes the rows' losses checks its arguments as the one without them does (no GPU needed)."""
import ctypes as C

from tests import abi


def test_arguments():
    L, f, nul, none = abi.lib(), C.c_float(1.0), None, abi.i64(-1)
    p = lambda v: C.c_void_p(v)
    good, ws = 1 << 20, C.c_size_t(1 << 40)

    def call(loss, dtype=0, n=3, dx=good, scale=f, workspace=good, size=ws):
        four = abi.i64(4)
        return L.gsb_linear_ce_grad_rows(p(good), dtype, four, abi.i64(n), p(good), four, abi.i64(9), four, p(good), none, scale, loss,
                                         p(good), nul, p(good), 1, nul, p(dx) if dx else nul, nul, p(workspace), size, nul, nul)

    assert call(p(good + 1)) == 1 and call(p(good + 2)) == 1
    assert call(p(good), dtype=7) == 1 and call(nul, dtype=7) == 1
    assert call(p(good), scale=C.c_float(float("inf"))) == 1
    assert call(p(good), dx=None) == 0                       # nothing is asked for
    assert call(p(good), size=C.c_size_t(0)) == 3            # a workspace too small
    assert call(p(good), n=0) == 0
