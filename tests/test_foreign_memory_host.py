"""Tensors over other allocators' memory: how long the owner is kept, and which memory is refused. No GPU: the
library's calls are played by the test, which says when an event has passed."""
import gc
import weakref

import pytest

import mantle_amd as m
from mantle_amd import _lib, tensor


class Owner:
    pass


class Played:
    """The library: events in the order of their records, done up to `passed`."""

    def __init__(self):
        self.made, self.records, self.passed, self.waits = 0, {}, 0, 0

    def __call__(self, name, *a):
        if name == "mh_event_create":
            self.made += 1
            a[0]._obj.value = self.made
        elif name == "mh_event_record":
            self.records[a[0]] = max(self.records.values(), default=0) + 1
        elif name == "mh_event_done":
            ev, wait, out = a
            if wait:
                self.waits += 1
                self.passed = max(self.passed, self.records[ev])
            out._obj.value = int(self.records[ev] <= self.passed)
        else:
            assert name in ("mh_init", "mh_sync"), name


@pytest.fixture
def played(monkeypatch):
    p = Played()
    monkeypatch.setattr(_lib, "call", p)
    monkeypatch.setattr(tensor, "_initialized", True)
    monkeypatch.setattr(tensor, "_queued", True)
    monkeypatch.setattr(tensor, "_held", tensor._Held())
    return p


def over(shape=(4, 8), ptr=4096):
    o = Owner()
    return m.Tensor.over(ptr, shape, o), weakref.ref(o)


def test_an_owner_outlives_its_tensor_until_sync(played):
    t, alive = over()
    i = m.IndexTensor.over(4096, (3,), alive())
    view = t.share()
    del t, i
    gc.collect()
    assert alive() is not None
    del view
    assert alive() is not None  # a queued call may still use the memory
    m.sync()
    assert alive() is None


def test_without_queued_calls_an_owner_goes_at_once(played, monkeypatch):
    monkeypatch.setattr(tensor, "_queued", False)
    t, alive = over()
    del t
    assert alive() is None


def test_leaving_the_queued_mode_waits(played):
    t, alive = over()
    del t
    m.init(0, asynchronous=False)
    assert alive() is None and tensor._queued is False


def test_owners_go_when_their_event_has_passed(played):
    n = tensor._Held._BATCH
    refs = []
    for _ in range(3 * n):
        t, alive = over()
        refs.append(alive)
        del t
    assert played.made == 2 and all(r() is not None for r in refs)
    played.passed = 2
    for _ in range(n):
        t, alive = over()
        refs.append(alive)
        del t
    assert not any(r() for r in refs[:2 * n]) and all(r() is not None for r in refs[2 * n:])
    played.passed = 4
    for _ in range(n):  # events are used again
        t, _ = over()
        del t
    over()
    assert played.made == 3 and played.waits == 0
    assert not any(r() for r in refs)


def test_large_memory_is_not_held_without_end(played):
    held = tensor._Held
    elements = 1 << 30  # 4 GiB
    refs = []
    for _ in range(8):
        t, alive = over((elements,))
        refs.append(alive)
        del t
        assert tensor._held.total <= held._MOST_BYTES + 4 * elements
    assert played.waits > 0 and refs[0]() is None and refs[-1]() is not None
    m.sync()
    assert not any(r() for r in refs) and tensor._held.total == 0


def test_many_batches_are_not_held_without_end(played):
    for _ in range((tensor._Held._MOST + 8) * tensor._Held._BATCH):
        t, _ = over()
        del t
    assert len(tensor._held.batches) <= tensor._Held._MOST and played.waits > 0


def test_after_a_shutdown_owners_go(played, monkeypatch):
    def refuses(name, *a):
        raise m.MantleHipError(_lib.ERR_NOT_INIT, name)
    refs = []
    monkeypatch.setattr(_lib, "call", refuses)
    for _ in range(tensor._Held._BATCH):
        t, alive = over()
        refs.append(alive)
        del t
    over()
    assert not any(r() for r in refs)


def test_memory_without_an_owner_is_not_held(played):
    t = m.Tensor.over(4096, (4,))
    del t
    assert not tensor._held.owners


def test_address_off_a_float_is_refused(played):
    for off in (1, 2, 3):
        with pytest.raises(m.MantleHipError) as e:
            m.Tensor.over(4096 + off, (4,))
        assert e.value.code == _lib.ERR_INVALID
    assert m.Tensor.over(4100, (4,)).ptr == 4100


def test_strided_owner_is_refused(played):
    class Strided:
        def __init__(self, whole, shape):
            self.whole, self.shape = whole, shape

        def is_contiguous(self):
            return self.whole

        def data_ptr(self):
            return 4096
    with pytest.raises(m.MantleHipError) as e:
        m.Tensor.over(4096, (6, 4), Strided(False, (6, 4)))
    assert e.value.code == _lib.ERR_INVALID
    m.Tensor.over(4096, (6, 4), Strided(True, (6, 4)))
    m.Tensor.over(4096, (4, 6), Strided(False, (6, 4)))  # the memory of a transposed view, as it lies
    m.Tensor.over(4096 + 96, (4,), Strided(False, (6, 4)))  # a part of it
