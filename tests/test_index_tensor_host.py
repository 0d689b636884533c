"""Calls that take floats refuse an IndexTensor before any device work. No GPU: the addresses are made up and every
call into the library fails the test."""
import pytest

import mantle_amd as m
from mantle_amd import _lib, ops


@pytest.fixture
def no_calls(monkeypatch):
    monkeypatch.setattr(m.tensor, "_initialized", True)

    def call(name, *args):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(_lib, "call", call)


def F(*shape):
    return m.Tensor.over(4096, shape)


def X(*shape):
    return m.IndexTensor.over(4096, shape)



S = (4, 6)
CALLS = {
    "fill": (lambda t: m.fill(t, 1.0), [S]),
    "elwise_transform": (lambda r, t: m.elwise_transform(m.OP.EXP, r, t), [S, S]),
    "elwise_pow": (lambda r, t: m.elwise_pow(r, t, 3), [S, S]),
    "elwise_op": (lambda r, a, b: m.elwise_op(m.OP.ADD, r, a, b), [S, S, S]),
    "accumulate_grad": (m.accumulate_grad, [S, S]),
    "tsum": (lambda t, r: m.tsum(t, -1, r), [S, (1,)]),
    "tmax": (lambda t, r: m.tmax(t, 0, r), [S, (1, 6)]),
    "tstd": (lambda t, r: m.tstd(t, -1, r), [S, (1,)]),
    "ADD": (lambda r, a, b: m.forward_op(m.OP.ADD, r, a, b), [S, S, S]),
    "POW": (lambda r, a, b: m.forward_op(m.OP.POW, r, a, b), [S, S, (1,)]),
    "SUM": (lambda r, a: m.forward_op(m.OP.SUM, r, a), [(1,), S]),
    "RELU": (lambda r, a: m.forward_op(m.OP.RELU, r, a), [S, S]),
    "FMA": (lambda r, a, b, c: ops.FMA.forward(r, a, b, c), [S, S, S, S]),
    "CLIP": (lambda r, a: m.forward_op(m.OP.CLIP, r, a, attributes={"min": 0.0, "max": 1.0}), [S, S]),
    "LEAKYRELU": (lambda r, a: m.forward_op(m.OP.LEAKYRELU, r, a, attributes={"negative_slope": 0.1}), [S, S]),
    "MUL backward": (lambda u, a, b, g: m.backward_op(0, m.OP.MUL, u, a, b, g), [S, S, S, S]),
    "POW backward": (lambda u, a, b, g: m.backward_op(0, m.OP.POW, u, a, b, g), [S, S, (1,), S]),
    "TANH backward": (lambda u, a, g: m.backward_op(0, m.OP.TANH, u, a, None, g), [S, S, S]),
    "MAX backward": (lambda u, a, g: m.backward_op(0, m.OP.MAX, u, a, None, g), [(1,), S, S]),
    "both of DIV": (lambda u, a, b, g, h: ops.backward_op_both(m.OP.DIV, u, a, b, g, h), [S] * 5),
    "both of POW": (lambda u, a, b, g, h: ops.backward_op_both(m.OP.POW, u, a, b, g, h), [S, S, (1,), S, (1,)]),
    "bias_relu": (m.bias_relu_forward, [S, S, S, (6,)]),
    "bias_relu backward": (lambda u, y, gx, gb, gy: m.bias_relu_backward(u, y, (6,), gx, gb, gy), [S, S, S, (6,), S]),
    "softmax": (m.softmax_forward, [S, S]),
    "softmax backward": (m.softmax_backward, [S, S, S]),
    "logsoftmax": (m.logsoftmax_forward, [S, S]),
    "logsoftmax backward": (m.logsoftmax_backward, [S, S, S]),
    "cross_entropy": (m.cross_entropy_forward, [(1,), S, S]),
    "cross_entropy backward": (m.cross_entropy_backward, [S, S, S, (1,)]),
    "softmax_log_mul_mean": (m.softmax_log_mul_mean_forward, [(1,), S, S]),
    "softmax_log_mul_mean backward": (m.softmax_log_mul_mean_backward, [S, S, S, (1,)]),
    "Adam": (lambda p, g: m.Adam([(p, g)]), [S, S]),
}


@pytest.mark.parametrize("name", CALLS)
def test_refused_in_every_place(no_calls, name):
    f, shapes = CALLS[name]
    for at in range(len(shapes)):
        with pytest.raises(m.MantleHipError) as e:
            f(*[(X if i == at else F)(*s) for i, s in enumerate(shapes)])
        assert e.value.code == _lib.ERR_INVALID, (name, at, e.value)
        assert "whole numbers" in str(e.value)


def test_refused_as_a_models_input_and_upper_gradient(no_calls):
    class Sym:
        class shape:
            num_elements = staticmethod(lambda: 24)
    with pytest.raises(m.MantleHipError) as e:
        m.Model._table([X(4, 6)], [Sym])
    assert e.value.code == _lib.ERR_INVALID
    assert m.Model._table([F(4, 6)], [Sym])[1] == _lib.FROM_DEVICE


def test_what_an_index_tensor_keeps(no_calls):
    t = X(3)
    assert t.ptr == 4096 and t.num_elements() == 3 and isinstance(t.share(), m.IndexTensor)
    with pytest.raises(AssertionError, match="mh_zero was called"):  # zero bits are the whole number 0
        t.zero()
    assert F(3).f32 == 4096


@pytest.mark.parametrize("make", [F, X])
def test_an_element_past_the_ends_is_refused(no_calls, make):
    t = make(2, 3)
    for i in (-1, 6, 1 << 40):
        with pytest.raises(IndexError):
            t[i]
        with pytest.raises(IndexError):
            t[i] = 1
    for i in (0, 5):
        with pytest.raises(AssertionError, match="mh_memcpy_d2h was called"):
            t[i]
        with pytest.raises(AssertionError, match="mh_memcpy_h2d was called"):
            t[i] = 1


def test_no_ids_at_all(monkeypatch):
    made = []
    monkeypatch.setattr(m.tensor, "_initialized", True)
    monkeypatch.setattr(_lib, "call", lambda name, *a: made.append(name))
    for none in ([], [[]]):
        t = m.IndexTensor.from_numpy(none)
        assert isinstance(t, m.IndexTensor) and t.num_elements() == 0
    assert "mh_memcpy_h2d" not in made
