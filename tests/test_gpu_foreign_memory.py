"""Tensors over another allocator's memory while calls are queued: dropped at once, their memory stays until the calls
are done, and is given back then."""
import weakref

import numpy as np
import pytest

from test_gpu_head import check, inputs, reference
from util import TEST_ASYNC, GpuEngine

pytestmark = pytest.mark.gpu


class Pool:
    """An allocator that hands a block out again, and lets it be written, when its owner is gone."""

    def __init__(self, m):
        self.m, self.free = m, []

    def take(self, a):
        m, pool = self.m, self

        class Block:
            def __init__(self):
                self.t = (m.IndexTensor if a.dtype == np.int32 else m.Tensor).from_numpy(a)

            def __del__(self):
                pool.free.append(self.t)
        return Block()


def queued(m):
    m.init(0, asynchronous=True)


def test_dropped_while_a_step_is_queued():
    m = GpuEngine().m
    x, w, labels = inputs(2048, 200, 9001, seed=51)
    want, bound = reference(x, w, labels)
    queued(m)
    try:
        pool = Pool(m)
        loss, one = m.Tensor(1), m.Tensor.from_numpy(np.float32([1]))
        gx, gw = m.Tensor(*x.shape), m.Tensor(*w.shape)
        m.sync()
        blocks = [pool.take(a) for a in (x, w, labels)]
        refs = [weakref.ref(b) for b in blocks]
        over = [(m.IndexTensor if a.dtype == np.int32 else m.Tensor).over(b.t.ptr, a.shape, b) for a, b in zip((x, w, labels), blocks)]
        m.linear_cross_entropy_step(loss, gx, gw, *over, one, accumulate=False)
        del over, blocks
        assert all(r() is not None for r in refs) and not pool.free
        m.sync()
        assert not any(r() for r in refs) and len(pool.free) == 3
        check({"loss": loss.to_numpy()[0], "grad_x": gx.to_numpy(), "grad_w": gw.to_numpy()}, want, bound, "dropped")
    finally:
        m.init(0, asynchronous=TEST_ASYNC)


def test_a_loop_that_makes_its_tensors_anew_gives_memory_back():
    m = GpuEngine().m
    queued(m)
    try:
        m.sync()
        block = m.Tensor.from_numpy(np.ones(64, np.float32))
        out = m.Tensor(64)
        n, refs = 3 * m.tensor._Held._BATCH, []

        class Owner:
            pass
        for _ in range(n):
            o = Owner()
            refs.append(weakref.ref(o))
            m.elwise_op(m.OP.ADD, out, m.Tensor.over(block.ptr, (64,), o), block)
        del o
        m._lib.call("mh_sync")  # not m.sync(), which lets go of all
        # the first of these closes the last batch; by the time that the next one closes its event has passed
        for _ in range(m.tensor._Held._BATCH + 2):
            m.Tensor.over(block.ptr, (64,), Owner())
            m._lib.call("mh_sync")
        assert not any(r() for r in refs)
        assert (out.to_numpy() == 2).all()
    finally:
        m.init(0, asynchronous=TEST_ASYNC)
