"""An Adam's largest norm is checked where it is set, before a step counts."""
import pytest

import mantle_amd as m
from mantle_amd import _lib


@pytest.fixture
def tensor(monkeypatch):
    """Tensors over made-up addresses, whose memory no call of these tests reaches."""
    monkeypatch.setattr(m.tensor, "_initialized", True)
    return lambda *shape: m.Tensor.over(4096, shape)


def refused(code, f):
    with pytest.raises(m.MantleHipError) as e:
        f()
    assert e.value.code == code, e.value


@pytest.mark.parametrize("bad", [-1.0, float("nan"), -float("inf"), -1e-45])
def test_refused_when_made(bad):
    refused(_lib.ERR_INVALID, lambda: m.Adam([], max_norm=bad))


class _Adam(m.Adam):
    """An optimizer over nothing, without memory of its own."""

    def __init__(self, norm, max_norm=None):
        self._collection = self._span = self.symbols = self._tables = None
        self.params, self.momentum_grads, self.rms_grads = [], [], []
        self.lr, self.beta1, self.beta2, self.epsilon, self.iter = 1e-3, 0.9, 0.999, 1e-8, 0
        self.max_norm, self.grad_norm = max_norm, norm


@pytest.mark.parametrize("bad", [-1.0, float("nan")])
def test_refused_when_set(tensor, bad):
    opt = _Adam(tensor(1), 1.0)
    with pytest.raises(m.MantleHipError) as e:
        opt.max_norm = bad
    assert e.value.code == _lib.ERR_INVALID and opt.max_norm == 1.0
    opt.max_norm = None
    opt.max_norm = 2
    assert opt.max_norm == 2.0


@pytest.mark.parametrize("shape", [(2,), (0,), (1, 3)])
def test_a_refused_step_does_not_count(tensor, shape):
    """A norm of more than one element, or of whole numbers."""
    for norm, code in ((tensor(*shape), _lib.ERR_SHAPE), (m.IndexTensor.over(4096, (1,)), _lib.ERR_INVALID)):
        opt = _Adam(norm, 1.0)
        refused(code, opt.step)
        assert opt.iter == 0
