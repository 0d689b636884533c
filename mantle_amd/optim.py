"""Adam over device-resident parameters: a mirror of mantle/nn/optim.mojo:51-149.

``Adam(params, lr, beta1, beta2, epsilon)`` takes a model's ``Parameters`` (its graph's
trainable parameters, get_trainable_parameters, optim.mojo:27-44) or (param, grad) ``Tensor``
pairs, and keeps
the momentum and rms tensors, zero-initialised, beside them. ``step()`` increments ``iter``
and updates every parameter with one ``mh_adam_step_multi`` launch per 80 tensors;
``zero_grad()`` zeroes the gradients (``Collection.set_zero``, collection.mojo:221-224).

``grad_norm`` and ``clip_grad_norm`` take the norm of many gradients together and scale them to
a largest one; an Adam with ``max_norm`` does so on their way into its step (no counterparts in
the reference).
"""
from __future__ import annotations

import ctypes
from array import array
from typing import List, Optional, Sequence, Tuple

from . import _lib
from .tensor import Tensor


class SymbolTensors(list):
    """Adam's momentum / rms tensors, one per parameter in order; indexable by position or, for
    an Adam built from a model's parameters, by the parameter's Symbol (as the reference's
    ``optim.momentum_grads[sym]`` collections are)."""

    def __init__(self, tensors, symbols=None):
        super().__init__(tensors)
        self.symbols = list(symbols) if symbols is not None else None

    def __getitem__(self, key):
        if self.symbols is not None and hasattr(key, "name") and hasattr(key, "shape"):
            return super().__getitem__(self.symbols.index(key))
        return super().__getitem__(key)


def _grad_tables(grads: Sequence[Tensor]):
    """The addresses and sizes of gradients, as the C ABI takes them."""
    n = len(grads)
    for kind in set(map(type, grads)):  # 400 tensors: 30 us, a property and a call each 75
        if kind is not Tensor:
            [g.f32 for g in grads]  # refuses whole numbers
    ptrs = array("Q", [g._ptr for g in grads])
    sizes = array("q", [g._shape._n for g in grads])
    return n, (ctypes.c_void_p * n).from_buffer(ptrs), (ctypes.c_int64 * n).from_buffer(sizes)


def _norm_address(norm: Optional[Tensor]):
    if norm is None:
        return None
    if norm.num_elements() != 1:
        raise _lib.MantleHipError(_lib.ERR_SHAPE, f"norm must hold one element (holds {norm.num_elements()})")
    return norm.f32


def grad_norm(norm: Tensor, grads: Sequence[Tensor]) -> None:
    """norm (one element) = the square root of the sum of the squares of every element of `grads`."""
    n, ptrs, sizes = _grad_tables(grads)
    _lib.call("mh_grad_norm", n, ptrs, sizes, _norm_address(norm))


def clip_grad_norm(norm: Optional[Tensor], grads: Sequence[Tensor], max_norm: float) -> None:
    """grad_norm, and every gradient scaled in place by min(1, max_norm / norm); none where one of their elements is
    infinite or NaN, as norm then shows. Tensors that share elements are refused."""
    n, ptrs, sizes = _grad_tables(grads)
    _lib.call("mh_clip_grad_norm", n, ptrs, sizes, float(max_norm), _norm_address(norm))


class Adam:
    def __init__(self, params, lr: float = 0.001, beta1: float = 0.9, beta2: float = 0.999,
                 epsilon: float = 1e-8, max_norm: Optional[float] = None):
        """``params``: a model's ``Parameters`` (its graph's trainable parameters, as
        ``Adam[g](model.parameters, ...)`` takes them), or (param, grad) Tensor pairs.
        ``max_norm``: each step takes the gradients scaled to at most this norm of all of them
        together, which ``self.grad_norm`` (one element, or None to go without) gets; the gradients
        themselves stay as they are."""
        self._collection = None
        self._span = None  # (params, grads, n) of a model's contiguous trainable span
        self.symbols = None  # the trainable parameters' symbols, for a model's parameters
        if hasattr(params, "tensors") and hasattr(params, "grads") and hasattr(params, "graph"):
            self._collection = params
            span = params.param_span()
            if span is not None:
                self._span = span
            self.symbols = params.graph.trainable_parameters()
            params = [(params.tensors[s], params.grads[s]) for s in self.symbols]
        self.params: List[Tuple[Tensor, Tensor]] = list(params)
        for p, g in self.params:
            if p.shape() != g.shape():
                raise _lib.MantleHipError(_lib.ERR_SHAPE, "a parameter and its gradient differ in shape")
            p.f32, g.f32  # neither holds whole numbers
        self.lr, self.beta1, self.beta2, self.epsilon = float(lr), float(beta1), float(beta2), float(epsilon)
        self.max_norm = max_norm
        self.grad_norm = None if max_norm is None else Tensor(1)
        self.iter = 0
        # allocate_rms_and_momentum (optim.mojo:142-149): zero-initialised, one per parameter;
        # over a model's span, two span-sized buffers whose slices are the per-parameter tensors
        if self._span is not None:
            _, _, n = self._span
            self._m_span, self._v_span = Tensor(n), Tensor(n)
            offs = [p.ptr - self._span[0] for p, _ in self.params]
            mom = [Tensor(p.shape(), _ptr=self._m_span.ptr + o, _owner=self._m_span)
                   for (p, _), o in zip(self.params, offs)]
            rms = [Tensor(p.shape(), _ptr=self._v_span.ptr + o, _owner=self._v_span)
                   for (p, _), o in zip(self.params, offs)]
        else:
            mom = [Tensor(p.shape()) for p, _ in self.params]
            rms = [Tensor(p.shape()) for p, _ in self.params]
        self.momentum_grads = SymbolTensors(mom, self.symbols)
        self.rms_grads = SymbolTensors(rms, self.symbols)
        self._tables = None  # step()'s pointer tables, with the tensors they were made from

    _max_norm: Optional[float] = None

    @property
    def max_norm(self) -> Optional[float]:
        return self._max_norm

    @max_norm.setter
    def max_norm(self, value: Optional[float]) -> None:
        if value is not None and not float(value) >= 0.0:
            raise _lib.MantleHipError(_lib.ERR_INVALID, f"a largest norm of {value}")
        self._max_norm = None if value is None else float(value)

    def zero_grad(self) -> None:
        """Adam.zero_grad (optim.mojo:90-92): parameters.grads.set_zero()."""
        if self._collection is not None:
            self._collection.grads.set_zero()
            return
        for _, g in self.params:
            g.zero()

    def step(self) -> None:
        norm = None if self.max_norm is None else _norm_address(self.grad_norm)
        self.iter += 1
        if self._span is not None:  # every parameter of the model in one launch
            p, g, n = self._span
            if self.max_norm is not None:
                one = [(ctypes.c_void_p * 1)(a) for a in (p, g, self._m_span.ptr, self._v_span.ptr)]
                _lib.call("mh_adam_clip_step_multi", 1, *one, (ctypes.c_int64 * 1)(n), self.lr, self.beta1, self.beta2,
                          self.epsilon, self.iter, self.max_norm, norm)
                return
            _lib.call("mh_adam_step", p, g, self._m_span.ptr, self._v_span.ptr, n, self.lr, self.beta1, self.beta2,
                      self.epsilon, self.iter)
            return
        n = len(self.params)
        if n == 0:
            if self.max_norm is not None and self.grad_norm is not None:
                self.grad_norm.zero()
            return
        # A tensor's address never changes, so the tables are made again only where a tensor was
        # exchanged (made on every step, those of 400 parameters cost as much as the step: 337 us
        # with them, 247 us without).
        made = (self.params, list(self.momentum_grads), list(self.rms_grads))
        if self._tables is None or self._tables[0] != made:
            VP = ctypes.c_void_p * n
            self._tables = ((list(made[0]), made[1], made[2]), VP(*[p.f32 for p, _ in self.params]),
                            VP(*[g.f32 for _, g in self.params]), VP(*[t.f32 for t in self.momentum_grads]),
                            VP(*[t.f32 for t in self.rms_grads]),
                            (ctypes.c_int64 * n)(*[p.num_elements() for p, _ in self.params]))
        _, ps, gs, ms, vs, sizes = self._tables
        if self.max_norm is not None:
            _lib.call("mh_adam_clip_step_multi", n, ps, gs, ms, vs, sizes, self.lr, self.beta1, self.beta2, self.epsilon,
                      self.iter, self.max_norm, norm)
            return
        _lib.call("mh_adam_step_multi", n, ps, gs, ms, vs, sizes, self.lr, self.beta1, self.beta2, self.epsilon,
                  self.iter)
