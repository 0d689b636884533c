"""Device-resident Tensor[f32] and TensorShape, mirroring mantle/core/tensor.mojo.

The reference keeps tensors in host memory (``Tensor`` allocates with ``alloc`` and zero-fills,
tensor.mojo:250-302). Here the storage is HBM on the initialised gfx950 device
(``mh_malloc`` + a zero-fill kernel); host copies are explicit (``from_numpy`` /
``to_numpy``), so chains of ops never cross PCIe.
"""
from __future__ import annotations

import ctypes
import functools
import math
from collections import deque
from typing import Iterable, Optional, Tuple, Union

import numpy as np

from . import _lib

MAX_RANK = _lib.MAX_RANK

_initialized = False
_queued = False  # calls return before their work is done


def init(device: int = 0, asynchronous: bool = False) -> None:
    """Initialise the library on `device` (idempotent)."""
    global _initialized, _queued
    _lib.call("mh_init", int(device), _lib.INIT_ASYNC if asynchronous else 0)
    _initialized = True
    if _queued and not asynchronous:
        sync()
    _queued = bool(asynchronous)


def ensure_init() -> None:
    if not _initialized:
        init(0)


def sync() -> None:
    _lib.call("mh_sync")
    _held.clear()


class _Held:
    """Owners of other allocators' memory whose tensors are gone while queued calls may still use it. They are let go
    when an event behind those calls has passed: one for _BATCH owners, or for _BATCH_BYTES of larger ones, so that a
    loop that makes its tensors anew on each pass pays for an event every thirty passes or so (one every 256 MB made a
    pass of 62 us over 246 MB one of 65), and waits for none unless _MOST batches or _MOST_BYTES are still held."""
    _BATCH, _LARGE, _BATCH_BYTES = 256, 1 << 20, 4 << 30
    _MOST, _MOST_BYTES = 64, 16 << 30

    def __init__(self):
        self.owners, self.bytes = [], 0  # bytes: of the large ones
        self.batches, self.total = deque(), 0  # (event, owners, bytes); the bytes of all of them
        self.events = []

    def large(self, nbytes: int) -> None:
        self.bytes += nbytes
        if self.bytes >= self._BATCH_BYTES:
            self.close()

    def close(self) -> None:
        try:
            if not self.events:
                p = ctypes.c_void_p()
                _lib.call("mh_event_create", ctypes.byref(p))
                self.events.append(p.value)
            _lib.call("mh_event_record", self.events[-1])
        except _lib.MantleHipError as e:
            if e.code != _lib.ERR_NOT_INIT:
                raise
            self.clear()  # shut down, which has waited for every call
            return
        ev, owners, nbytes = self.events.pop(), self.owners[:], self.bytes
        del self.owners[:len(owners)]
        self.bytes = 0
        self.batches.append((ev, owners, nbytes))
        self.total += nbytes
        done = ctypes.c_int()
        while self.batches:
            ev, _, nbytes = self.batches[0]
            wait = len(self.batches) > 1 and (len(self.batches) > self._MOST or self.total > self._MOST_BYTES)
            _lib.call("mh_event_done", ev, int(wait), ctypes.byref(done))
            if not done.value:
                break
            self.batches.popleft()
            self.total -= nbytes
            self.events.append(ev)

    def clear(self) -> None:
        """Everything queued is done."""
        self.owners.clear()
        self.bytes = 0
        while self.batches:
            self.events.append(self.batches.popleft()[0])
        self.total = 0


_held = _Held()


class TensorShape:
    """Row-major shape of rank 1..8 (tensor.mojo:28-229)."""

    __slots__ = ("_dims", "_n", "_cs")

    def __init__(self, *dims: Union[int, Iterable[int]]):
        if len(dims) == 1 and not isinstance(dims[0], (int, np.integer)):
            dims = tuple(dims[0])
        d = dims
        for x in dims:  # plain ints, as nearly always, are taken as they are
            if type(x) is not int:
                d = tuple(map(int, dims))
                break
        if not 1 <= len(d) <= MAX_RANK:
            raise ValueError(f"rank {len(d)} outside 1..{MAX_RANK}")
        self._dims = d
        self._n = math.prod(d)
        self._cs = None

    def __getstate__(self):
        """The dims alone; what is made from them is made again, so older pickles load too."""
        return None, {"_dims": self._dims}

    def __setstate__(self, state) -> None:
        self.__init__(*state[1]["_dims"])

    def rank(self) -> int:
        return len(self._dims)

    def num_elements(self) -> int:
        return self._n

    def strides(self) -> Tuple[int, ...]:  # tensor.mojo:143-155
        st, s = [], 1
        for x in reversed(self._dims):
            st.append(s)
            s *= x
        return tuple(reversed(st))

    @property
    def dims(self) -> Tuple[int, ...]:
        return self._dims

    def __getitem__(self, i: int) -> int:
        return self._dims[i]

    def __len__(self) -> int:
        return len(self._dims)

    def __eq__(self, other) -> bool:
        if isinstance(other, TensorShape):
            return self._dims == other._dims
        if isinstance(other, tuple):
            return self._dims == other
        return NotImplemented

    def __hash__(self):
        return hash(self._dims)

    def __repr__(self) -> str:
        return "TensorShape(" + ", ".join(str(x) for x in self._dims) + ")"

    def c(self) -> _lib.mh_shape:
        """The shape as the C ABI takes it (read during the call), made once: a shape never changes,
        and the four of a binary gradient's call cost more to make than its launch."""
        if self._cs is None:
            self._cs = _lib.make_shape(self._dims)
        return self._cs


def as_shape(s) -> TensorShape:
    return s if isinstance(s, TensorShape) else TensorShape(s)


# A shape is the same object every time its dims come from a tuple: a loop over tensors of other allocators' makes
# eight of them on each pass of a few calls, and half of its time.
_shape_of = functools.lru_cache(maxsize=1024)(TensorShape)


class Tensor:
    """fp32 tensor in device memory. ``share()`` aliases, ``copy()`` deep-copies
    (tensor.mojo:345-393)."""

    __slots__ = ("_shape", "_ptr", "_owner", "_foreign", "__weakref__")

    def __init__(self, *shape, _ptr: Optional[int] = None, _owner=None):
        ensure_init()
        self._foreign = 0  # 1 + the bytes of another allocator's memory with an owner
        self._shape = as_shape(shape[0]) if len(shape) == 1 and not isinstance(shape[0], (int, np.integer)) \
            else TensorShape(*shape)
        if _ptr is not None:
            self._ptr, self._owner = _ptr, _owner
            return
        p = ctypes.c_void_p()
        n = self._shape.num_elements()
        _lib.call("mh_malloc", ctypes.byref(p), max(n, 1) * 4)
        self._ptr, self._owner = p.value, None
        _lib.call("mh_zero", self._ptr, n)  # zero-initialised, tensor.mojo:266, 284

    def __del__(self):
        try:
            if self._foreign:
                if _queued:
                    _held.owners.append(self._owner)
                    if self._foreign > _Held._LARGE:
                        _held.large(self._foreign)
            elif self._owner is None and self._ptr:
                _lib.lib().mh_free(self._ptr)
                self._ptr = None
        except Exception:
            pass  # not made whole, or the library is shut down and has waited for every call

    @classmethod
    def over(cls, ptr: int, shape, owner=None) -> "Tensor":
        """A tensor over device memory that another allocator holds: row-major, 4 bytes an element and aligned
        to them. What wrote that memory has to be done: the library works on a stream of its own. `owner` is kept
        alive with the tensor and, where calls are queued, until those that were queued while the tensor lived are
        done; that shows at a sync(), or when tensors like this one come and go. Without an owner the memory has
        to outlast those calls (sync() waits for them)."""
        if not _initialized:
            init(0)
        if len(_held.owners) >= _Held._BATCH:
            _held.close()
        t = cls.__new__(cls)
        t._foreign = 0
        t._owner = 0  # anything but None: not freed here
        t._shape = _shape_of(shape) if type(shape) is tuple else as_shape(shape)
        t._ptr = ptr = int(ptr)
        if ptr & 3:
            raise _lib.MantleHipError(_lib.ERR_INVALID, f"address {ptr:#x} is not aligned to 4 bytes")
        if owner is not None:
            try:
                whole = owner.is_contiguous()
            except (AttributeError, TypeError):  # not an array that could be strided
                whole = True
            if not whole and owner.data_ptr() == ptr and tuple(owner.shape) == t._shape._dims:
                raise _lib.MantleHipError(_lib.ERR_INVALID, "the owner's elements do not lie one after another")
            t._owner, t._foreign = owner, 4 * t._shape._n + 1
        return t

    # ---- properties ----
    def shape(self) -> TensorShape:
        return self._shape

    def num_elements(self) -> int:
        return self._shape.num_elements()

    def rank(self) -> int:
        return self._shape.rank()

    def dim(self, i: int) -> int:
        return self._shape[i]

    @property
    def ptr(self) -> int:
        return self._ptr

    @property
    def f32(self) -> int:
        """The address, for a call that takes floats there."""
        return self._ptr

    # ---- host transfer ----
    @staticmethod
    def from_numpy(a) -> "Tensor":
        a = np.ascontiguousarray(a, dtype=np.float32)
        t = Tensor(TensorShape(a.shape if a.ndim else (1,)))
        if a.size:
            _lib.call("mh_memcpy_h2d", t._ptr, a.ctypes.data, a.size * 4)
        return t

    def to_numpy(self) -> np.ndarray:
        out = np.empty(self._shape.dims, dtype=np.float32)
        if out.size:
            _lib.call("mh_memcpy_d2h", out.ctypes.data, self._ptr, out.size * 4)
        return out

    # ---- tensor.mojo API ----
    def copy(self) -> "Tensor":
        t = Tensor(self._shape)
        _lib.call("mh_memcpy_d2d", t._ptr, self._ptr, self.num_elements() * 4)
        return t

    def share(self) -> "Tensor":
        return Tensor(self._shape, _ptr=self._ptr, _owner=self)

    def zero(self) -> None:
        _lib.call("mh_zero", self._ptr, self.num_elements())

    def _at(self, i: int) -> int:
        """The address of element i, counted over all dims."""
        i = int(i)
        if not 0 <= i < self._shape._n:
            raise IndexError(f"element {i} of {self}")
        return self._ptr + 4 * i

    def __getitem__(self, i: int) -> float:
        v = np.empty(1, dtype=np.float32)
        _lib.call("mh_memcpy_d2h", v.ctypes.data, self._at(i), 4)
        return float(v[0])

    def __setitem__(self, i: int, val: float) -> None:
        v = np.array([val], dtype=np.float32)
        _lib.call("mh_memcpy_h2d", self._at(i), v.ctypes.data, 4)

    def __repr__(self) -> str:
        return f"Tensor({self._shape})"


class IndexTensor(Tensor):
    """int32 tensor in device memory: class labels, chosen ids and counts. The reference holds these
    as one-hot float tensors (loss.mojo:45-61), which a large vocabulary rules out. The calls that take floats
    refuse it."""

    __slots__ = ()

    @property
    def f32(self) -> int:
        raise _lib.MantleHipError(_lib.ERR_INVALID, f"{self} holds whole numbers where the call takes floats")

    @staticmethod
    def from_numpy(a) -> "IndexTensor":
        a = np.asarray(a)
        if a.size and (a.dtype.kind not in "iub" or a.max() > 0x7fffffff or a.min() < -0x80000000):
            raise ValueError(f"ids are whole numbers of 32 bits, not {a.dtype}")
        a = np.ascontiguousarray(a, dtype=np.int32)
        t = IndexTensor(TensorShape(a.shape if a.ndim else (1,)))
        if a.size:
            _lib.call("mh_memcpy_h2d", t._ptr, a.ctypes.data, a.size * 4)
        return t

    def to_numpy(self) -> np.ndarray:
        out = np.empty(self._shape.dims, dtype=np.int32)
        if out.size:
            _lib.call("mh_memcpy_d2h", out.ctypes.data, self._ptr, out.size * 4)
        return out

    def copy(self) -> "IndexTensor":
        t = IndexTensor(self._shape)
        _lib.call("mh_memcpy_d2d", t._ptr, self._ptr, self.num_elements() * 4)
        return t

    def share(self) -> "IndexTensor":
        return IndexTensor(self._shape, _ptr=self._ptr, _owner=self)

    def __getitem__(self, i: int) -> int:
        v = np.empty(1, dtype=np.int32)
        _lib.call("mh_memcpy_d2h", v.ctypes.data, self._at(i), 4)
        return int(v[0])

    def __setitem__(self, i: int, val: int) -> None:
        v = np.array([val], dtype=np.int32)
        _lib.call("mh_memcpy_h2d", self._at(i), v.ctypes.data, 4)

    def __repr__(self) -> str:
        return f"IndexTensor({self._shape})"
