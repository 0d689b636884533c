"""The router over more rows than its workgroups take at once: each goes round two times or more with the same LDS, in
the forward (1024 workgroups) and in the backward (2048), by sorted lists and by rounds of a maximum. Bounds are those of
test_gpu_router.py."""
import numpy as np
import pytest

from test_gpu_router import check, inputs, m_, reference, run

pytestmark = pytest.mark.gpu

SIZES = [(70000, 64, 6), (70000, 64, 12), (9000, 600, 10), (5000, 1024, 8), (5000, 1000, 40), (40000, 200, 9), (300000, 7, 3), (150001, 30, 9)]


@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_rounds(size, normalise):
    print(f"\n[router] {size} {normalise}", flush=True)
    x, keep, gw = inputs(*size, seed=71)
    m = m_()
    want = reference(x, size[2], keep, normalise, gw, 0.3)
    check(run(m, x, size[2], keep, normalise, gw, 0.3), *want, what=str(size))
    g = np.random.RandomState(0).standard_normal(x.shape).astype(np.float32)
    got = run(m, x, size[2], keep, normalise, gw, 0.3, grad=g)["grad_x"]
    assert np.array_equal(got, g + run(m, x, size[2], keep, normalise, gw, 0.3)["grad_x"])


def test_a_kept_row_without_an_expert_shows():
    """Every logit at minus infinity: a softmax over nothing. The row's weights and the loss are NaN, as its probabilities
    are; its choices stay in range, and other rows are what they are alone."""
    x, keep, gw = inputs(50, 24, 4, seed=72)
    keep[:] = 1
    x[9] = -np.inf
    for normalise in (False, True):
        got = run(m_(), x, 4, keep, normalise, gw, 1.0)
        assert np.isnan(got["loss"]) and np.isnan(got["weights"][9]).all() and np.isnan(got["grad_x"][9]).all()
        assert sorted(got["chosen"][9]) == [0, 1, 2, 3]
        assert np.isfinite(np.delete(got["weights"], 9, 0)).all() and np.isfinite(np.delete(got["grad_x"], 9, 0)).all()
        keep[9] = 0  # left out, it counts nowhere
        want = reference(np.where(keep[:, None] != 0, x, 0.0).astype(np.float32), 4, keep, normalise, gw, 1.0)
        check(run(m_(), x, 4, keep, normalise, gw, 1.0), *want, what="left out")
        keep[9] = 1
