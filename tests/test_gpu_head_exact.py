"""How exact the vocabulary head's cross entropy is where elements differ widely in size.

The bounds are those of test_gpu_head.py with what an element far below the largest is off by: x and w are held as
two halves, the largest element in [2^14, 2^15), so that fp16's least step of 2^-24 leaves at most 2^-39 of the largest:
of its row's in x for the logits, of the tensor's (for x: of the kept rows') otherwise. Up to 64 rows (128 forward)
against a large w three bf16 an element have no such floor, but for grad_w."""
import numpy as np
import pytest

from test_gpu_head import U, inputs, m_, run

pytestmark = pytest.mark.gpu
FLOOR = 2.0 ** -39


def reference(x, w, labels, ug=1.0):
    """The results in 64 bits and the bounds of their errors."""
    labels = labels.astype(np.int64)
    keep = labels >= 0
    x, w = np.where(keep[:, None], x, 0.0).astype(np.float64), w.astype(np.float64)
    n = max(1, int(keep.sum()))
    rows, dim = x.shape
    classes = w.shape[0]
    z = x @ w.T
    top = z.max(1, keepdims=True)
    e = np.exp(z - top)
    logsum = np.log(e.sum(1))
    lse = top[:, 0] + logsum
    at = np.arange(rows), np.maximum(labels, 0)
    row = np.where(keep, logsum - (z[at] - top[:, 0]), 0.0)
    p = e / e.sum(1, keepdims=True)
    g = p.copy()
    g[at] -= 1.0
    g *= keep[:, None]
    c = ug / n

    def product(k):
        return 2.0 ** -21 + (3 * k / 16 + 8) * 2 * U

    ax, aw, ag = np.abs(x), np.abs(w), np.abs(g)
    bz = (ax @ aw.T) * product(dim) + FLOOR * (ax.max(1)[:, None] * aw.sum(1)[None] + aw.max() * ax.sum(1)[:, None]) + U * np.abs(z)
    # errors of the logits move the log-sum-exp by their mean over p, those of the sums by their own
    bs = (128 + classes / 512 + 40) * U
    bl = (p * bz).sum(1) + bz.max(1) * (p * bz).sum(1) + bs + 4 * U * np.abs(lse)
    brow = bl + bz[at] + 4 * U * (np.abs(lse) + np.abs(z[at]))
    return {"z": z, "p": p, "row_loss": row, "row_lse": np.where(keep, lse, 0.0), "loss": row.sum() / n,
            "grad_x": c * (g @ w), "grad_w": c * (g.T @ x)}, \
        {"row_loss": brow * keep, "row_lse": bl * keep, "loss": (brow * keep).sum() / n + 4 * U * abs(row.sum() / n)}, \
        (bz, bl, ag, ax, aw, abs(c), product, keep)


def gradient_bounds(want, parts, rounding):
    """Bounds of the gradients from an element of G's: p times what its exponent is off by, `rounding` more of p, and G's halves."""
    bz, bl, ag, ax, aw, c, product, keep = parts
    dg = (want["p"] * (bz + bl[:, None] + rounding) + 2.0 ** -22 * ag + 2.0 ** -40) * keep[:, None]
    floor_x = FLOOR * aw.max() * ag.sum(1)[:, None]
    floor_w = FLOOR * ax.max() * ag.sum(0)[:, None]
    return {"grad_x": c * (dg @ aw + (ag @ aw) * product(aw.shape[0] + 256) + floor_x) + 4 * U * np.abs(want["grad_x"]),
            "grad_w": c * (dg.T @ ax + (ag.T @ ax) * product(ax.shape[0] + 256) + floor_w) + 4 * U * np.abs(want["grad_w"])}


def check(got, want, bound, what=""):
    for k in bound:
        if k in got:
            off = np.abs(got[k].astype(np.float64) - want[k])
            over = ~(off <= bound[k] + 1e-42)
            assert not over.any(), f"{what} {k}: {over.sum()} of {over.size} beyond the bound, worst {np.max(off - bound[k]):.3g}"


SIZES = [(130, 64, 1000), (300, 200, 2049), (9, 300, 16390)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_a_row_does_not_depend_on_the_size_of_others(size):
    """Every other row 2^26 times the size: what it leaves of the others' bits is what they have alone."""
    x, w, labels = inputs(*size, seed=31, left_out=0)
    x[::2] *= np.float32(2.0 ** 26)
    for how in ("step", "two calls"):
        got = run(m_(), x, w, labels, how=how)
        check(got, *reference(x, w, labels)[:2], what=f"{size} {how}")
    one = run(m_(), np.ascontiguousarray(x[1::2]), w, np.ascontiguousarray(labels[1::2]), how="two calls")
    assert np.array_equal(one["row_lse"], got["row_lse"][1::2]) and np.array_equal(one["row_loss"], got["row_loss"][1::2])


@pytest.mark.parametrize("spread", [20, 24, 28])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_columns_of_different_sizes(size, spread):
    """Column k of x times 2^s_k and of w times 2^-s_k: every product as it was, every operand spread."""
    x, w, labels = inputs(*size, seed=32)
    s = np.random.RandomState(33).randint(-spread // 2, spread // 2 + 1, size[1])
    x, w = np.ldexp(x, s).astype(np.float32), np.ldexp(w, -s).astype(np.float32)
    want, bound, parts = reference(x, w, labels)
    bound.update(gradient_bounds(want, parts, 2.0 ** -21 + 8 * U * (np.abs(want["z"]) + np.abs(want["row_lse"])[:, None])))
    for how in ("step", "two calls"):
        check(run(m_(), x, w, labels, how=how), want, bound, what=f"{size} {how}")


@pytest.mark.parametrize("where", ["x", "w", "both"])
def test_single_outliers(where):
    """One element 2^18 times the others, in a row that is kept or in a class."""
    for size in SIZES:
        x, w, labels = inputs(*size, seed=34)
        labels[5] = 7
        if where != "w":
            x[5, 3] = 2.0 ** 18
        if where != "x":
            w[11, 8] = -2.0 ** 18
        want, bound, parts = reference(x, w, labels)
        bound.update(gradient_bounds(want, parts, 2.0 ** -21 + 8 * U * (np.abs(want["z"]) + np.abs(want["row_lse"])[:, None])))
        for how in ("step", "two calls"):
            check(run(m_(), x, w, labels, how=how), want, bound, what=f"{size} {how}")


OFFSETS = [((5, 40, 300), 30000.0), ((200, 70, 3000), -1000.0), ((7, 260, 17000), 30000.0), ((70, 300, 14100), 4000.0)]


def with_offset(size, offset, seed):
    """Inputs whose logits all lie near `offset`: a column of ones in x, of the offset in w."""
    x, w, labels = inputs(*size, seed=seed, left_out=0)
    x[:, 0], w[:, 0] = 1.0, offset
    return x, w, labels


@pytest.mark.parametrize("size, offset", OFFSETS, ids=str)
def test_gradient_rows_add_up_to_zero(size, offset):
    """sum_v G_nv = 0, whatever the log-sum-exp's size: column 0 of grad_x is offset times it. An element of G is off by
    2^-22 of itself or 2^-40; a row of probabilities by its sums' roundings, those of 1 / sum and the product with it
    (4 U in all), and by an exponential's, which the sum takes with another instruction: (3 |z - top| + 8) U each. The
    product has its own bound."""
    x, w, labels = with_offset(size, offset, 35)
    want, _, parts = reference(x, w, labels)
    ag, aw, product = parts[2], parts[4], parts[6]
    away = want["z"].max(1)[:, None] - want["z"]
    rows = (want["p"] * (3 * away + 8)).sum(1) * U + (128 + size[2] / 512 + 44) * U
    tol = 2.0 ** -22 * ag.sum(1) + size[2] * 2.0 ** -40 + rows + ag.sum(1) * product(size[2] + 256)
    for how in ("step", "two calls"):
        g = run(m_(), x, w, labels, how=how)["grad_x"][:, 0].astype(np.float64) * size[0] / offset
        assert (np.abs(g) <= tol).all(), f"{how}: {np.max(np.abs(g) / tol)} of the bound"
        if size[2] < 1000:  # below what a log-sum-exp rounded to fp32 does; a long product's bound is above that
            assert (tol < 2.0 ** -24 * abs(offset) / 4).all()


@pytest.mark.parametrize("size, offset", OFFSETS, ids=str)
def test_loss_of_logits_with_an_offset(size, offset):
    """A row's loss is the difference of two logits, each rounded to U of itself beside its product's error, and a
    logarithm; nothing of it is rounded at the size of the log-sum-exp. A logit near the offset is a sum of one large
    product, exact but for its operands' (a power of two times a whole number holds in a half), and small ones."""
    x, w, labels = with_offset(size, offset, 36)
    w[:, 0] = np.ldexp(1.0, int(np.log2(abs(offset))))  # exact in one half
    want, _, parts = reference(x, w, labels)
    at = np.arange(size[0]), labels
    small = np.abs(x[:, 1:].astype(np.float64)) @ np.abs(w[:, 1:].astype(np.float64)).T
    k = size[1]
    # small products' halves, floors, and the sum's additions at the size of the offset (truncating: 2 U each)
    bz = small * 2.0 ** -21 + FLOOR * (np.abs(x).max(1)[:, None] * np.abs(w.astype(np.float64)).sum(1)[None]
                                       + np.abs(w).max() * np.abs(x.astype(np.float64)).sum(1)[:, None]) \
        + (3 * k / 16 + 2) * 2 * U * np.abs(want["z"])
    tol = 2 * bz.max(1) + (128 + size[2] / 512 + 48) * U + 4 * U * want["row_loss"]
    got = run(m_(), x, w, labels, how="two calls")
    assert (np.abs(got["row_loss"] - want["row_loss"]) <= tol).all()
