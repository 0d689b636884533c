"""Scores far below fp32's least, and a weight's last bits (group_router_forward), against the formulas in 64 bits.

Tolerances, U = 2^-24. Scores and their sums are 64-bit to 2^-30 of themselves or better, so a weight is one
rounding, 1.1 U of itself."""
import numpy as np
import pytest

from test_gpu_group_router import inputs, m_, reference, run

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def check(a, what=""):
    a = dict(a, scale=float(np.float32(a["scale"])))  # as the call has it
    got, (want, _, whole) = run(m_(), **a), reference(**a)
    for k, v in whole.items():
        assert np.array_equal(got[k], v), f"{what} {k}"
    off = np.abs(got["weights"] - want["weights"])
    assert (off <= 1.1 * U * np.abs(want["weights"]) + 1e-44).all(), f"{what}: weights off by {(off / np.abs(want['weights']).clip(1e-44)).max() / U} U"


def small(rows, experts, k, scores, seed):
    d = inputs(rows, experts, k, seed=seed)
    del d["gw"]
    r = np.random.RandomState(seed + 1)
    if scores == "sigmoid":
        d["x"] = (d["x"] - r.choice([0.0, 85.0, 90.0, 100.0, 115.0, 300.0, 600.0], (rows, 1))).astype(np.float32)
        d["bias"] = None
    else:  # the likely experts are shut
        d["x"][:, ::2] -= r.choice([0.0, 85.0, 95.0, 110.0, 300.0, 600.0], (rows, 1)).astype(np.float32)
        d["bias"] = np.where(np.arange(experts) % 2, -np.inf, 0.0).astype(np.float32)
    return d


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("rows, experts, k, groups, opened", [(60, 16, 2, 1, 1), (70, 60, 5, 6, 3), (33, 300, 20, 1, 1), (2500, 16, 2, 4, 2),
                                                              (2300, 60, 20, 1, 1), (2100, 256, 8, 8, 4), (2100, 1024, 6, 1, 1)])
def test_scores_below_the_least_float(rows, experts, k, groups, opened, scores):
    """Choices among scores of down to e^-600, which add up to less than fp32 holds: the weights are their shares all the same."""
    d = small(rows, experts, k, scores, seed=rows + experts)
    check(dict(d, groups=groups, keep_groups=opened, scores=scores, normalise=True, scale=2.5), "normalised")
    # not normalised: scores that fp32 holds with few bits, but not times the scale
    check(dict(d, groups=groups, keep_groups=opened, scores=scores, normalise=False, scale=1e30), "scaled")


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("rows, experts, k", [(50, 7, 3), (500, 60, 5), (3000, 60, 8), (2100, 256, 8), (2050, 1000, 12)])
def test_last_bits(rows, experts, k, scores, normalise):
    d = inputs(rows, experts, k, seed=rows + k, std=0.1 if scores == "sigmoid" else 0.5 / experts)
    d["x"] *= np.float32(4.0)
    del d["gw"]
    check(dict(d, scores=scores, normalise=normalise, scale=1.5))
