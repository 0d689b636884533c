"""Scores far below fp32's least, and the gradient's last bits (group_router_*), against the formulas in 64 bits.

Tolerances, U = 2^-24. Scores, their sums and the sums of g s are 64-bit to 2^-30 of themselves or better, so a weight is one
rounding, 1.1 U of itself, and a gradient of a chosen expert 1.1 U and 2^-28 of s (|g| + sum |g| q), which a difference of gradients
may leave nothing of. Under a softmax that is not normalised every expert has one: an exponential is off by an ulp of the unit's, 2 U,
and U / 4 for its argument, and so are their sum and sum g q; with a rounding of the factor and one of the product 7 U of s (|g| +
sum |g| q), the |g| the chosen's own."""
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
    if "gw" in a:
        # s (|g| + sum |g| q) of each expert, from a reference of gradients that add up
        x, k, kept = a["x"].astype(np.float64), a["k"], whole["chosen"] >= 0
        sel = np.where(kept, whole["chosen"], 0)
        at = np.arange(len(x))[:, None]
        if a["scores"] == "sigmoid":
            e = np.exp(-np.abs(x))
            s, rest = np.where(x < 0, e, 1) / (1 + e), np.where(x < 0, 1, e) / (1 + e)
        else:
            s = np.exp(x - x.max(1, keepdims=True))
            s, rest = s / s.sum(1, keepdims=True), np.ones_like(x)
        q = s[at, sel] / (s[at, sel].sum(1, keepdims=True) if a["normalise"] else 1)
        g = np.abs(a["gw"].astype(np.float64))
        size = np.zeros_like(x)
        if a["scores"] == "softmax" and not a["normalise"]:
            size += s * (g * q).sum(1, keepdims=True)
        size[at, sel] = q * rest[at, sel] * (g + (g * q).sum(1, keepdims=True))
        off = np.abs(got["grad_x"] - want["grad_x"])
        size *= abs(a["scale"]) * kept[:, :1]
        every = a["scores"] == "softmax" and not a["normalise"]
        bound = 1e-44 + (7 * U * size if every else 1.1 * U * np.abs(want["grad_x"]) + 2.0 ** -28 * size)
        over = ~(off <= bound)
        assert not over.any(), f"{what}: {over.sum()} gradients off, the worst {(off / bound.clip(1e-44)).max()} bounds"


def small(rows, experts, k, scores, seed):
    d = inputs(rows, experts, k, seed=seed)
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
    """Choices among scores of down to e^-600, which add up to less than fp32 holds: the weights are their shares all the same, and
    have the formula's gradient."""
    d = small(rows, experts, k, scores, seed=rows + experts)
    check(dict(d, groups=groups, keep_groups=opened, scores=scores, normalise=True, scale=2.5), "normalised")
    # not normalised: scores that fp32 holds with few bits, but not times the scale
    d["gw"] = (d["gw"] * 1e-20).astype(np.float32)
    check(dict(d, groups=groups, keep_groups=opened, scores=scores, normalise=False, scale=1e30), "scaled")


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("rows, experts, k", [(50, 7, 3), (500, 60, 5), (3000, 60, 8), (2100, 256, 8), (2050, 1000, 12)])
def test_last_bits(rows, experts, k, scores, normalise):
    d = inputs(rows, experts, k, seed=rows + k, std=0.1 if scores == "sigmoid" else 0.5 / experts)
    d["x"] *= np.float32(4.0)
    check(dict(d, scores=scores, normalise=normalise, scale=1.5))
