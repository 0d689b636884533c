"""Refusals of the norm, the grouped router, the gradients' norm and sampling, which need no GPU: every argument is checked
before any device work. An address in these calls is never read."""
import ctypes

import pytest

import mantle_amd as m
from mantle_amd import _lib

P = ctypes.c_void_p(4096)
I, O, N, S, OK = _lib.ERR_INVALID, _lib.ERR_OVERFLOW, _lib.ERR_NULL, _lib.ERR_SHAPE, _lib.OK
NAN, INF = float("nan"), float("inf")


@pytest.fixture
def tensor(monkeypatch):
    """Tensors over made-up addresses: the checks of shapes and kinds come before the library's."""
    monkeypatch.setattr(m.tensor, "_initialized", True)
    return lambda *shape: m.Tensor.over(4096, shape), lambda *shape: m.IndexTensor.over(4096, shape)


def refused(code, f, *args, **kw):
    with pytest.raises(m.MantleHipError) as e:
        f(*args, **kw)
    assert e.value.code == code, e.value


@pytest.mark.parametrize("rows, dim, eps, code", [(-1, 4, 0, I), (4, 0, 0, I), (4, -1, 0, I), (4, 4, -1e-9, I), (4, 4, NAN, I), (4, 4, INF, I),
                                                  (4, (1 << 30) + 1, 0, O), (1 << 20, 1 << 27, 0, O)])
def test_norm_sizes(rows, dim, eps, code):
    L = _lib.lib()
    assert L.mh_rms_norm_fwd(P, P, P, P, P, rows, dim, eps) == code
    assert L.mh_rms_norm_bwd(P, P, P, P, P, P, rows, dim, eps, 0) == code


def test_norm_null():
    L = _lib.lib()
    for hole in (0, 2, 4):  # out, x, w
        assert L.mh_rms_norm_fwd(*[None if i == hole else P for i in range(5)], 4, 4, 0) == N, hole
    for hole in (2, 4, 5):  # grad_out, h, w
        assert L.mh_rms_norm_bwd(*[None if i == hole else P for i in range(6)], 4, 4, 0, 0) == N, hole
    assert L.mh_rms_norm_bwd(None, None, P, P, P, P, 4, 4, 0, 0) == OK  # nothing is asked for
    assert L.mh_rms_norm_fwd(None, None, None, None, None, 0, 4, 0) == OK
    assert L.mh_rms_norm_bwd(P, None, None, None, None, None, 0, 4, 0, 0) == OK


# rows, experts, k, groups, open groups, best, scores, scale
@pytest.mark.parametrize("a, code", [((-1, 4, 2, 1, 1, 2, 1, 1), I), ((4, 0, 1, 1, 1, 2, 1, 1), I), ((4, 4, 0, 1, 1, 2, 1, 1), I), ((4, 4, 5, 1, 1, 2, 1, 1), I),
                                     ((4, 1025, 2, 1, 1, 2, 1, 1), I), ((4, 1024, 65, 1, 1, 2, 1, 1), I), ((1 << 30, 4, 2, 1, 1, 2, 1, 1), O),
                                     ((4, 8, 2, 0, 1, 2, 1, 1), I), ((4, 8, 2, 3, 1, 2, 1, 1), I), ((4, 8, 2, 4, 0, 2, 1, 1), I), ((4, 8, 2, 4, 5, 2, 1, 1), I),
                                     ((4, 8, 3, 4, 1, 2, 1, 1), I), ((4, 128, 2, 128, 4, 1, 1, 1), I), ((4, 8, 2, 4, 2, 0, 1, 1), I),
                                     ((4, 8, 2, 4, 2, 3, 1, 1), I), ((4, 8, 2, 4, 2, 2, 2, 1), I), ((4, 8, 2, 4, 2, 2, -1, 1), I),
                                     ((4, 8, 2, 4, 2, 2, 1, NAN), I), ((4, 8, 2, 4, 2, 2, 1, INF), I)])
def test_group_router_sizes(a, code):
    L = _lib.lib()
    rows, experts, k, groups, opened, best, scores, scale = a
    assert L.mh_group_router_fwd(P, P, P, P, P, P, rows, experts, k, groups, opened, best, scores, 1, scale) == code
    if (groups, opened, best) == (1, 1, 2) or scores not in (0, 1) or scale != 1:
        assert L.mh_group_router_bwd(P, P, P, P, P, rows, experts, k, scores, 1, scale, 0) == code


def test_group_router_null():
    L = _lib.lib()
    for hole in range(4):  # weights, chosen, counts, x
        assert L.mh_group_router_fwd(*[None if i == hole else P for i in range(6)], 4, 8, 2, 4, 2, 2, 1, 1, 1) == N, hole
    for hole in (0, 1, 3, 4):
        assert L.mh_group_router_bwd(*[None if i == hole else P for i in range(5)], 4, 8, 2, 1, 1, 1, 0) == N, hole
    assert L.mh_group_router_bwd(None, None, None, None, None, 0, 8, 2, 1, 1, 1, 0) == OK
    for experts, rate, code in ((0, 1, I), (1025, 1, I), (4, NAN, I), (4, INF, I)):
        assert L.mh_router_bias_update(P, P, experts, rate) == code
    assert L.mh_router_bias_update(None, P, 4, 1) == N and L.mh_router_bias_update(P, None, 4, 1) == N


def table(*sizes, hole=None, base=4096):
    n = len(sizes)
    return n, (ctypes.c_void_p * n)(*[None if i == hole else base + (i << 40) for i in range(n)]), (ctypes.c_int64 * n)(*sizes)


def test_gradient_norm():
    L = _lib.lib()
    n, ptrs, sizes = table(5, 7)
    adam = lambda n, g, s, top=1.0, iter=1: L.mh_adam_clip_step_multi(n, ptrs, g, ptrs, ptrs, s, 0.1, 0.9, 0.99, 1e-8, iter, top, P)  # noqa: E731
    for call in (lambda n, g, s: L.mh_grad_norm(n, g, s, P), lambda n, g, s: L.mh_clip_grad_norm(n, g, s, 1.0, P), adam):
        assert call(-1, ptrs, sizes) == I
        assert call(2, None, sizes) == N and call(2, ptrs, None) == N
        assert call(*table(5, -1)) == I
        assert call(*table(5, 7, hole=1)) == N
        assert call(*table(5, 7, base=4098)) == I  # no address of floats
        assert call(*table(1 << 46, 1)) == O
    assert L.mh_grad_norm(n, ptrs, sizes, None) == N
    for top in (-1.0, NAN, -INF):
        assert L.mh_clip_grad_norm(n, ptrs, sizes, top, P) == I
        assert adam(n, ptrs, sizes, top) == I
    assert adam(n, ptrs, sizes, iter=0) == I


def test_tensors_that_share_elements_are_refused():
    L = _lib.lib()
    at = lambda *a: (ctypes.c_void_p * len(a))(*a)  # noqa: E731
    size = lambda *a: (ctypes.c_int64 * len(a))(*a)  # noqa: E731
    for ptrs, sizes in ((at(4096, 4096), size(1, 1)), (at(4096, 4132), size(10, 2)), (at(8192, 4096), size(4, 1025)),
                        (at(4096, 9000, 4100), size(1, 5, 1226))):
        assert L.mh_clip_grad_norm(len(ptrs), ptrs, sizes, 1.0, P) == I
        assert b"shares" in L.mh_last_error()
    for ptrs, sizes in ((at(4096, 4096), size(0, 1)), (at(4096, 4136), size(10, 2)), (at(8192, 4096), size(4, 1024))):
        L.mh_clip_grad_norm(len(ptrs), ptrs, sizes, -1.0, P)
        assert b"shares" not in L.mh_last_error()


@pytest.mark.parametrize("rows, classes, code", [(-1, 4, I), (4, 0, I), (4, (1 << 24) + 1, O), (1 << 31, 4, O)])
def test_sample_sizes(rows, classes, code):
    assert _lib.lib().mh_sample_tokens(P, P, P, P, P, P, P, P, rows, classes) == code


def test_sample_null():
    L = _lib.lib()
    for hole in (0, 2, 3):  # tokens, x, u
        assert L.mh_sample_tokens(*[None if i == hole else P for i in range(8)], 4, 4) == N, hole
    assert L.mh_sample_tokens(*[None] * 8, 0, 4) == OK


def test_shapes_and_kinds(tensor):
    F, X = tensor
    norm = [F(3, 4), F(3, 4), F(4)]
    for at, t, code in [(0, F(4, 3), S), (0, X(3, 4), I), (1, X(3, 4), I), (1, F(3, 5), S), (2, F(5), S), (2, X(4), I), (2, None, I)]:
        refused(code, m.rms_norm_forward, *[t if i == at else a for i, a in enumerate(norm)])
    refused(S, m.rms_norm_forward, *norm, residual=F(4))
    refused(I, m.rms_norm_forward, *norm, sum=X(3, 4))
    back = [F(3, 4), F(4), F(3, 4), F(3, 4), F(4)]
    for at, t, code in [(0, F(3, 5), S), (1, F(3, 4), S), (1, X(4), I), (2, None, I), (2, F(4), S), (3, X(3, 4), I), (4, F(3), S)]:
        refused(code, m.rms_norm_backward, *[t if i == at else a for i, a in enumerate(back)])
    refused(S, m.rms_norm_backward, *back, grad_sum=F(3))
    rf = [F(6, 2), X(6, 2), X(8), F(6, 8)]
    for at, t, code in [(0, F(6, 3), S), (1, X(5, 2), S), (1, F(6, 2), I), (2, X(9), S), (2, F(8), I), (3, F(8), S)]:
        refused(code, m.group_router_forward, *[t if i == at else a for i, a in enumerate(rf)])
    refused(S, m.group_router_forward, *rf, bias=F(9))
    refused(I, m.group_router_forward, *rf, bias=X(8))
    refused(S, m.group_router_forward, *rf, keep=X(7))
    refused(I, m.group_router_forward, *rf, scores="tanh")
    refused(I, m.group_router_forward, *rf, groups=3)
    refused(I, m.group_router_forward, *rf, groups=4, keep_groups=5)
    refused(S, m.group_router_backward, F(6, 8), F(6, 8), X(6, 2), F(6, 1))
    refused(I, m.group_router_backward, F(6, 8), F(6, 8), X(6, 2), F(6, 2), scores="")
    refused(S, m.router_bias_update, F(7), X(8), 0.1)
    refused(I, m.router_bias_update, F(8), F(8), 0.1)
    sm = [X(6), F(6, 9), F(6)]
    for at, t, code in [(0, X(7), S), (0, F(6), I), (1, F(6), S), (1, X(6, 9), I), (2, F(5), S)]:
        refused(code, m.sample_tokens, *[t if i == at else a for i, a in enumerate(sm)])
    for kw in ({"temperature": F(5)}, {"top_k": X(5)}, {"top_p": F(1)}, {"min_p": F(6, 1)}, {"logprob": F(7)}):
        refused(S, m.sample_tokens, *sm, **kw)
    refused(I, m.sample_tokens, *sm, top_k=F(6))
    refused(S, m.grad_norm, F(2), [F(3)])
    refused(I, m.grad_norm, X(1), [F(3)])
    refused(I, m.grad_norm, F(1), [F(3), X(3)])
    refused(I, m.clip_grad_norm, F(1), [F(3)], -1.0)
    refused(I, m.clip_grad_norm, F(1), [F(3), F(3)], 1.0)  # one tensor twice
