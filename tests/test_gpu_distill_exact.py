"""Distillation where logits are large: masked teachers, logits with an offset, the backward alone. Bounds are those of
test_gpu_distill.py at the size of the logits' differences."""
import numpy as np
import pytest

from test_gpu_distill import check, inputs, m_, reference, run

pytestmark = pytest.mark.gpu
LOWEST = -3.4028234663852886e38
SIZES = [(5, 40, 3), (3, 1000, 8), (40, 3001, 9), (7, 20000, 20), (300, 33000, 9), (3, 70001, 30), (258, 65541, 4)]


@pytest.mark.parametrize("T", [0.5, 1.0, 4.0])
def test_teacher_rows_of_the_lowest_value(T):
    """A teacher whose entries are all the type's lowest value says that they are alike; beside larger ones that they are
    none. Their quotient by T is no number of the type where T < 1."""
    x, ids, teacher = inputs(6, 500, 7, seed=41, left_out=0)
    teacher[1] = LOWEST
    teacher[2, 3:] = LOWEST
    alike = teacher.copy()
    alike[1] = 0.0
    alike[2, 3:] = -1e6
    want, bound = reference(x, ids, alike, T=T)
    for how in ("step", "two calls"):
        check(run(m_(), x, ids, teacher, T=T, how=how), want, bound, how)


def with_offset(size, seed, offset=4096.0):
    """Logits on a grid of 2^-10, and the same with the offset, which fp32 holds exactly."""
    x, ids, teacher = inputs(*size, seed=seed, left_out=0.0 if size[0] < 4 else 0.1)
    x = (np.round(x * 1024) / 1024).astype(np.float32)
    moved = (x + np.float32(offset)).astype(np.float32)
    assert np.array_equal(moved.astype(np.float64) - offset, x)
    return x, moved, ids, teacher


@pytest.mark.parametrize("offset", [4096.0, -4096.0])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_loss_of_logits_with_an_offset(size, offset):
    """The loss does not change, nor does its bound: one row at a time, a mean would hide a row's rounding."""
    x, moved, ids, teacher = with_offset(size, 42, offset)
    rows = np.flatnonzero((ids >= 0).any(1))[:3]
    for T in (1.0, 2.5):
        for r in rows:
            one = slice(r, r + 1)
            want, bound = reference(x[one], ids[one], teacher[one], T=T)
            got = run(m_(), moved[one], ids[one], teacher[one], T=T)
            off = abs(float(got["loss"]) - want["loss"])
            assert off <= bound["loss"], (r, T, off, bound["loss"])
        want, bound = reference(x, ids, teacher, T=T)
        off = abs(float(run(m_(), moved, ids, teacher, T=T)["loss"]) - want["loss"])
        assert off <= bound["loss"], (T, off, bound["loss"])


@pytest.mark.parametrize("how", ["step", "two calls"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_gradient_of_logits_with_an_offset(size, how):
    """Neither the gradient nor its bound changes, in the backward alone as in the step, accumulated too."""
    for offset in (4096.0, -4096.0):
        x, moved, ids, teacher = with_offset(size, 43, offset)
        g = np.random.RandomState(0).standard_normal(x.shape).astype(np.float32)
        for T in (1.0, 2.5):
            want, bound = reference(x, ids, teacher, T=T)
            got = run(m_(), moved, ids, teacher, T=T, how=how)["grad_x"]
            check({"grad_x": got}, want, bound, f"{how} {offset} {T}")
            assert np.array_equal(run(m_(), moved, ids, teacher, T=T, how=how, grad=g)["grad_x"], g + got)


@pytest.mark.parametrize("T", [0.5, 1.0])
@pytest.mark.parametrize("size", [(3, 500, 4), (2, 40001, 9), (3, 131072, 5), (300, 70001, 6)], ids=str)
def test_rows_all_at_the_lowest_value(size, T):
    """A student whose logits are all the type's lowest value has every class at 1 / classes."""
    x, ids, teacher = inputs(*size, seed=44, left_out=0)
    x[1] = 0.0
    want, bound = reference(x, ids, teacher, T=T)
    x[1] = LOWEST
    for how in ("step", "two calls"):
        got = run(m_(), x, ids, teacher, T=T, how=how)
        check({"grad_x": got["grad_x"], "loss": got["loss"]}, want, bound, how)
