"""The C entry points with outputs that begin in the middle of a buffer (a flat gradient buffer, say), and dropout
in place: the same bits as with outputs of their own, and nothing written beside them."""
import ctypes as C

import pytest
import torch

from tests import abi

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
F, NEG = C.c_float(1.0), abi.i64(-1)


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def inside(n, dt, off):
    """n elements that begin `off` elements behind a 16-byte boundary, in a buffer of marks."""
    whole = torch.full((n + 64,), 7.0, dtype=dt, device="cuda")
    return whole, whole[32 + off:32 + off + n]


def untouched(whole, off, n):
    return bool((whole[:32 + off] == 7).all()) and bool((whole[32 + off + n:] == 7).all())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(200, 300, 64), (130, 40, 100), (150, 2100, 72), (90, 300, 128), (100, 300, 200), (70, 300, 264), (300, 60, 36)])
@pytest.mark.parametrize("off", [1, 2, 4])
def test_gradients_into_the_middle_of_a_buffer(gsb, dt, N, V, D, off):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(N, D, device="cuda", generator=g).to(dt)
    w = (torch.randn(V, D, device="cuda", generator=g) * D ** -0.5).to(dt)
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    L, code = abi.lib(), CODE[dt]
    sizes = (abi.i64(N), abi.ptr(w), abi.i64(D), abi.i64(V), abi.i64(D))
    loss, lse = torch.empty(N, device="cuda"), torch.empty(N, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    pull = torch.empty(N, D, device="cuda") if L.gsb_linear_ce_has_pull(code, abi.i64(V), abi.i64(D)) else None
    ws = torch.empty(L.gsb_linear_ce_workspace_bytes(code, abi.ptr(w), abi.i64(D), abi.i64(N), abi.i64(V), abi.i64(D),
                                                     int(pull is not None)), dtype=torch.uint8, device="cuda")
    abi.check(L.gsb_linear_ce(abi.ptr(x), code, abi.i64(D), *sizes, abi.ptr(t), NEG, F, abi.ptr(loss), abi.ptr(lse), abi.ptr(pull),
                              abi.ptr(ws), C.c_size_t(ws.numel()), abi.ptr(err), stream()), "gsb_linear_ce")
    ws = torch.empty(L.gsb_linear_ce_grad_workspace_bytes(code, abi.ptr(w), abi.i64(D), abi.i64(N), abi.i64(V), abi.i64(D),
                                                          int(pull is not None), 1, 1), dtype=torch.uint8, device="cuda")
    up = torch.randn(N, device="cuda", generator=g)

    def grads(dx, dw):
        abi.check(L.gsb_linear_ce_grad(abi.ptr(x), code, abi.i64(D), *sizes, abi.ptr(t), NEG, F, abi.ptr(lse), abi.ptr(pull),
                                       abi.ptr(up), 1, None, abi.ptr(dx), abi.ptr(dw), abi.ptr(ws), C.c_size_t(ws.numel()),
                                       abi.ptr(err), stream()), "gsb_linear_ce_grad")
        torch.cuda.synchronize()

    want_dx, want_dw = torch.empty_like(x), torch.empty_like(w)
    grads(want_dx, want_dw)
    all_x, dx = inside(N * D, dt, off)
    all_w, dw = inside(V * D, dt, off)
    grads(dx, dw)
    assert torch.equal(dx.view(N, D), want_dx) and torch.equal(dw.view(V, D), want_dw)
    assert untouched(all_x, off, N * D) and untouched(all_w, off, V * D) and int(err) == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [1, 100, 4099, 5000000, 40000001])
@pytest.mark.parametrize("off", [0, 1])
def test_dropout_in_place(gsb, dt, n, off):
    whole, x = inside(n, dt, off)
    x.copy_(torch.randn(n, device="cuda"))
    want = gsb.ops.dropout(x.clone(), 0.3, seed=4, stream=5)
    abi.check(abi.lib().gsb_dropout(abi.ptr(x), CODE[dt], abi.i64(n), C.c_double(0.3), C.c_uint64(4), C.c_uint32(5), None, abi.ptr(x),
                                    stream()), "gsb_dropout")
    torch.cuda.synchronize()
    assert torch.equal(x, want) and untouched(whole, off, n)
