"""Refusals of the language-model losses, which need no GPU: every argument is checked before any device
work. An address in these calls is never read."""
import ctypes

import pytest

import mantle_amd as m
from mantle_amd import _lib

P = ctypes.c_void_p(4096)
I, O, N, OK = _lib.ERR_INVALID, _lib.ERR_OVERFLOW, _lib.ERR_NULL, _lib.OK


@pytest.fixture
def tensor(monkeypatch):
    """Tensors over made-up addresses: the checks of shapes and kinds come before the library's."""
    monkeypatch.setattr(m.tensor, "_initialized", True)
    return lambda *shape: m.Tensor.over(4096, shape), lambda *shape: m.IndexTensor.over(4096, shape)


@pytest.mark.parametrize("sizes, code", [((-1, 4, 4), I), ((4, 0, 4), I), ((4, 4, 0), I), ((4, -1, 4), I), ((1 << 31, 4, 4), O),
                                         ((4, 4, 1 << 31), O), ((4, (1 << 24) + 1, 4), O), ((4, 1 << 24, 1 << 24), O)])
def test_head_sizes(sizes, code):
    L = _lib.lib()
    assert L.mh_linear_cross_entropy_fwd(P, P, P, P, P, P, *sizes) == code
    assert L.mh_linear_cross_entropy_bwd(P, P, P, P, P, P, P, *sizes, 1) == code
    assert L.mh_linear_cross_entropy_step(P, P, P, P, P, P, P, P, *sizes, 1) == code
    assert b"mh_linear_cross_entropy_step" in L.mh_last_error()


def test_head_null():
    L = _lib.lib()
    s = (4, 4, 4)
    for hole in (0, 3, 4, 5):  # loss, x, w, labels
        args = [None if i == hole else P for i in range(6)]
        assert L.mh_linear_cross_entropy_fwd(*args, *s) == N, hole
    for hole in (2, 3, 4, 5, 6):
        args = [None if i == hole else P for i in range(7)]
        assert L.mh_linear_cross_entropy_bwd(*args, *s, 0) == N, hole
    for hole in (0, 4, 5, 6, 7):
        args = [None if i == hole else P for i in range(8)]
        assert L.mh_linear_cross_entropy_step(*args, *s, 0) == N, hole
    assert L.mh_linear_cross_entropy_bwd(None, None, P, P, P, P, P, *s, 0) == OK  # nothing is asked for


@pytest.mark.parametrize("sizes, T, code", [((-1, 4, 2), 1, I), ((4, 0, 2), 1, I), ((4, 4, 0), 1, I), ((4, 4, 1025), 1, I),
                                            ((4, 4, 2), 0, I), ((4, 4, 2), -1, I), ((4, 4, 2), float("nan"), I),
                                            ((4, 4, 2), float("inf"), I), ((4, 4, 2), 1e-7, I), ((4, 4, 2), 2e6, I),
                                            ((4, 1 << 31, 2), 1, O), ((1 << 22, 4, 2), 1, O)])
def test_distill_sizes(sizes, T, code):
    L = _lib.lib()
    assert L.mh_distill_fwd(P, P, P, P, P, *sizes, T) == code
    assert L.mh_distill_bwd(P, P, P, P, P, P, *sizes, T, 1) == code
    assert L.mh_distill_step(P, P, P, P, P, P, P, *sizes, T, 1) == code


def test_distill_null():
    L = _lib.lib()
    for hole in (0, 2, 3, 4):
        assert L.mh_distill_fwd(*[None if i == hole else P for i in range(5)], 4, 4, 2, 1) == N, hole
    for hole in range(6):
        assert L.mh_distill_bwd(*[None if i == hole else P for i in range(6)], 4, 4, 2, 1, 0) == N, hole
    for hole in (0, 2, 3, 4, 5, 6):
        assert L.mh_distill_step(*[None if i == hole else P for i in range(7)], 4, 4, 2, 1, 0) == N, hole


@pytest.mark.parametrize("sizes, code", [((-1, 4, 2), I), ((4, 0, 1), I), ((4, 4, 0), I), ((4, 4, 5), I), ((4, 1025, 2), I),
                                         ((4, 1024, 65), I), ((1 << 30, 4, 2), O)])
def test_router_sizes(sizes, code):
    L = _lib.lib()
    assert L.mh_router_fwd(P, P, P, P, P, None, *sizes, 0) == code
    assert L.mh_router_bwd(P, P, None, P, P, P, P, *sizes, 0, 0) == code


def test_router_null():
    L = _lib.lib()
    for hole in range(5):
        assert L.mh_router_fwd(*[None if i == hole else P for i in range(6)], 4, 4, 2, 0) == N, hole
    for hole in (0, 1, 3, 4):
        assert L.mh_router_bwd(*[None if i == hole else P for i in range(7)], 4, 4, 2, 0, 0) == N, hole


def refused(code, f, *args, **kw):
    with pytest.raises(m.MantleHipError) as e:
        f(*args, **kw)
    assert e.value.code == code, e.value


def test_shapes_and_kinds(tensor):
    F, X = tensor
    S = _lib.ERR_SHAPE
    head = [F(1), F(6, 4), F(9, 4), F(6, 4), F(9, 4), X(6), F(1)]
    bad = [(0, F(2), S), (1, F(6, 5), S), (2, F(9, 5), S), (3, F(6), S), (3, F(6, 5), S), (4, F(9, 5), S), (5, X(7), S),
           (5, F(6), I), (5, None, I), (6, F(2), S), (6, None, I), (0, X(1), I)]
    for at, t, code in bad:
        refused(code, m.linear_cross_entropy_step, *[t if i == at else a for i, a in enumerate(head)])
    refused(S, m.linear_cross_entropy_forward, F(1), F(7), F(6, 4), F(9, 4), X(6))
    refused(S, m.linear_cross_entropy_backward, F(6, 4), F(9, 4), F(6, 4), F(9, 4), X(6), F(5), F(1))
    dis = [F(1), F(6, 9), F(6, 9), X(6, 2), F(6, 2), F(1)]
    for at, t, code in [(0, F(2), S), (1, F(6, 8), S), (2, F(5, 9), S), (3, X(6), S), (3, F(6, 2), I), (4, F(6, 3), S), (5, F(3), S)]:
        refused(code, m.distill_step, *[t if i == at else a for i, a in enumerate(dis)])
    refused(S, m.distill_step, *dis, row_lse=F(5))
    rf = [F(6, 2), X(6, 2), X(9), F(1), F(6, 9)]
    for at, t, code in [(0, F(6, 3), S), (1, X(5, 2), S), (1, F(6, 2), I), (2, X(8), S), (3, F(2), S), (4, F(9), S)]:
        refused(code, m.router_forward, *[t if i == at else a for i, a in enumerate(rf)])
    refused(S, m.router_forward, *rf, keep=X(7))
    refused(I, m.router_forward, *rf, keep=F(6))
    refused(S, m.router_backward, F(6, 9), F(6, 9), X(6, 2), X(9), F(6, 1), F(1))


def test_index_tensor_takes_whole_numbers_only():
    for bad in ([1.5], [1 << 40], [-(1 << 31) - 1]):
        with pytest.raises(ValueError):
            m.IndexTensor.from_numpy(bad)
