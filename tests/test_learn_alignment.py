"""Pointers that are no multiple of their element's size, or a workspace's of 16 bytes, are refused before
anything is launched (no GPU is needed, and none is touched: every call here has one bad pointer)."""
import ctypes as C

import pytest

from tests import abi

GOOD, WS = 1 << 20, 1 << 40        # addresses that are never used
F, NEG = C.c_float(1.0), abi.i64(-1)


def p(v):
    return C.c_void_p(v)


def embedding(dt, at):
    return abi.lib().gsb_embedding(p(at["w"]), dt, abi.i64(4), abi.i64(9), abi.i64(4), p(at["idx"]), abi.i64(3), F, NEG,
                                   p(at["out"]), p(at["err"]), None)


def embedding_grad(dt, at):
    return abi.lib().gsb_embedding_grad(p(at["w"]), dt, abi.i64(4), p(at["idx"]), abi.i64(3), abi.i64(9), F, NEG, p(at["out"]),
                                        p(at["ws"]), C.c_size_t(WS), p(at["err"]), None)


def embedding_sort(dt, at):
    return abi.lib().gsb_embedding_sort(p(at["idx"]), abi.i64(3), abi.i64(9), abi.i64(4), NEG, p(at["ids"]), p(at["num"]),
                                        p(at["ws"]), C.c_size_t(WS), p(at["err"]), None)


def embedding_rows(dt, at):
    return abi.lib().gsb_embedding_grad_rows(p(at["w"]), dt, abi.i64(4), abi.i64(3), abi.i64(9), abi.i64(2), F, p(at["out"]),
                                             p(at["ws"]), C.c_size_t(WS), None)


def dropout(dt, at):
    return abi.lib().gsb_dropout(p(at["w"]), dt, abi.i64(5), C.c_double(0.5), C.c_uint64(1), C.c_uint32(1), p(at["step"]),
                                 p(at["out"]), None)


def loss(dt, at):
    return abi.lib().gsb_linear_ce(p(at["x"]), dt, abi.i64(4), abi.i64(3), p(at["w"]), abi.i64(4), abi.i64(9), abi.i64(4),
                                   p(at["idx"]), NEG, F, p(at["loss"]), p(at["lse"]), None, p(at["ws"]), C.c_size_t(WS),
                                   p(at["err"]), None)


def total(dt, at):
    return abi.lib().gsb_linear_ce_total(p(at["loss"]), p(at["idx"]), NEG, abi.i64(9), abi.i64(3), 1, p(at["total"]),
                                         p(at["count"]), p(at["ws"]), C.c_size_t(WS), None)


def loss_grad(dt, at):
    return abi.lib().gsb_linear_ce_grad(p(at["x"]), dt, abi.i64(4), abi.i64(3), p(at["w"]), abi.i64(4), abi.i64(9), abi.i64(4),
                                        p(at["idx"]), NEG, F, p(at["lse"]), p(at["pull"]), p(at["up"]), 1, p(at["count"]),
                                        p(at["out"]), p(at["dw"]), p(at["ws"]), C.c_size_t(WS), p(at["err"]), None)


TYPED = {"w", "x", "out", "dw"}
WIDTHS = dict(idx=8, ids=8, num=8, step=8, err=4, loss=4, lse=4, pull=4, up=4, count=4, total=4, ws=16)
CALLS = [(embedding, ["w", "idx", "out", "err"]), (embedding_grad, ["w", "idx", "out", "ws", "err"]),
         (embedding_sort, ["idx", "ids", "num", "ws", "err"]), (embedding_rows, ["w", "out", "ws"]),
         (dropout, ["w", "step", "out"]), (loss, ["x", "w", "idx", "loss", "lse", "ws", "err"]),
         (total, ["loss", "idx", "total", "count", "ws"]),
         (loss_grad, ["x", "w", "idx", "lse", "pull", "up", "count", "out", "dw", "ws", "err"])]


@pytest.mark.parametrize("dt,size", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("call,names", CALLS, ids=[c.__name__ for c, _ in CALLS])
def test_a_pointer_off_its_elements_is_refused(call, names, dt, size):
    for name in names:
        width = size if name in TYPED else WIDTHS[name]
        for off in (1, width // 2):
            at = {n: GOOD for n in list(TYPED) + list(WIDTHS)}
            at[name] = GOOD + off
            assert call(dt, at) == 1, (name, off)
