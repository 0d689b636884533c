"""Distillation from a teacher's top logits (distill_*) against the formulas in 64 bits.

Tolerances, from the arithmetic, U = 2^-24 half a step of fp32: the exponent t = x log2(e) / T takes a factor of
three roundings, a multiply-add and the instruction's own step: e^y is off by (3 |t| + 4) U of itself. A log-sum-exp
is off by the mean of that over p, the roundings of its sums (C / 1024 a thread, 20 in the tree), of max / T
(twice) and of its own; p by its own exponent's and the log-sum-exp's; q, over k entries, likewise."""
import numpy as np
import pytest

from util import GpuEngine

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NONE = -1


def m_():
    return GpuEngine().m


def reference(x, ids, teacher, T=1.0, ug=1.0):
    ids = ids.astype(np.int64)
    with np.errstate(invalid="ignore"):
        there = (ids >= 0) & (teacher > -np.inf)
    some = there.any(1)
    n = max(1, int(some.sum()))
    x, t64 = np.where(some[:, None], x, 0.0).astype(np.float64), np.where(there, teacher, 0.0).astype(np.float64) / T
    rows, classes = x.shape
    r = np.arange(rows)[:, None]
    y = x / T
    top = y.max(1)
    lse = top + np.log(np.exp(y - top[:, None]).sum(1))
    p = np.exp(y - lse[:, None])
    u = np.where(there, t64, -1e300)
    best = u.max(1)
    logq = u - best[:, None] - np.log(np.exp(u - best[:, None]).sum(1, keepdims=True))
    q = np.where(there, np.exp(logq), 0.0)
    at = np.maximum(ids, 0)
    picked = y[r, at]
    live = there & (q > 0)
    with np.errstate(invalid="ignore"):
        inner = np.where(live, q * (logq - picked + lse[:, None]), 0.0)
    loss = T * T / n * inner.sum()
    c = ug * T / n
    spread = np.zeros_like(x)
    np.add.at(spread, (np.broadcast_to(r, at.shape), at), q)
    grad = c * (p - spread) * some[:, None]
    # bounds
    t = np.minimum(top[:, None] - y, 1e6) * 1.4427
    bl = U * ((p * (3 * t + 4)).sum(1) + classes / 1024 + 24 + 4 * np.abs(top) + 2 * np.abs(lse))
    bp = p * ((3 * t + 8) * U + bl[:, None] + 3 * U * (np.minimum(np.abs(y), 1e6) + np.abs(lse)[:, None]))
    size, best = np.abs(t64), np.where(some, np.abs(best), 0.0)[:, None]
    bq = q * U * (4 * size + 4 * best + ids.shape[1] / 512 + 40)
    with np.errstate(invalid="ignore"):
        bound_in = bq * (np.abs(np.maximum(logq, -1e6)) + np.abs(picked) + np.abs(lse)[:, None] + 1) \
            + q * (bl[:, None] + U * (4 * size + 4 * best + 4 * np.abs(picked) + 2 * np.abs(lse)[:, None] + 8))
    bound_in = np.where(live, bound_in, 0.0)
    dq = np.zeros_like(x)
    np.add.at(dq, (np.broadcast_to(r, at.shape), at), bq)
    bg = abs(c) * (bp + dq + 4 * U * (p + spread)) * some[:, None]
    out = {"loss": loss, "row_lse": np.where(some, lse, 0.0), "grad_x": grad}
    bound = {"loss": T * T / n * bound_in.sum() + (30 + ids.shape[1] / 512) * U * T * T / n * np.abs(inner).sum(),
             "row_lse": bl * some, "grad_x": bg}
    return out, bound


def inputs(rows, classes, k, seed, left_out=0.1, repeat=False):
    r = np.random.RandomState(seed)
    x = (2 * r.standard_normal((rows, classes))).astype(np.float32)
    teacher = -np.sort(-(2 * r.standard_normal((rows, k)) + 4), 1).astype(np.float32)
    if repeat or k > classes:
        ids = r.randint(0, max(1, min(classes, 5)), (rows, k)).astype(np.int32)
    else:
        ids = np.stack([r.choice(classes, k, replace=False) for _ in range(rows)]).astype(np.int32)
    ids[r.uniform(size=ids.shape) < left_out] = NONE
    ids[r.uniform(size=rows) < left_out] = -100
    return x, ids, teacher


def run(m, x, ids, teacher, T=1.0, ug=1.0, how="step", grad=None):
    rows, classes = x.shape
    tx, ti, tt, tu = m.Tensor.from_numpy(x), m.IndexTensor.from_numpy(ids), m.Tensor.from_numpy(teacher), m.Tensor.from_numpy(np.float32([ug]))
    loss, lse = m.Tensor(1), m.Tensor(rows)
    gx = m.Tensor.from_numpy(np.full(x.shape, 7.0, np.float32) if grad is None else grad)
    if how == "step":
        m.distill_step(loss, gx, tx, ti, tt, tu, temperature=T, row_lse=lse, accumulate=grad is not None)
    else:
        m.distill_forward(loss, lse, tx, ti, tt, temperature=T)
        m.distill_backward(gx, tx, ti, tt, lse, tu, temperature=T, accumulate=grad is not None)
    return {"loss": loss.to_numpy()[0], "row_lse": lse.to_numpy(), "grad_x": gx.to_numpy()}


def check(got, want, bound, what=""):
    for k, v in got.items():
        off = np.abs(v.astype(np.float64) - want[k])
        assert np.isfinite(v).all(), f"{what} {k}: not finite"
        over = off > bound[k] + 1e-38
        assert not over.any(), f"{what} {k}: {over.sum()} of {over.size} beyond the bound, worst {off.max():.3g} of {np.max(bound[k]):.3g}"


SIZES = [(1, 1, 1), (3, 2, 1), (1, 3, 3), (5, 7, 2), (16, 1000, 8), (33, 257, 64), (7, 4096, 100), (9, 4099, 65),
         (300, 1023, 5), (2, 32768, 17), (3, 32771, 128), (520, 33001, 3), (4, 70001, 256), (1, 131072, 1024), (513, 8191, 12), (300, 70003, 9)]


@pytest.mark.parametrize("how", ["step", "two calls"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, how):
    print(f"\n[distill] {size} {how}", flush=True)
    a = inputs(*size, seed=sum(size), left_out=0.0 if size[0] < 4 else 0.1)
    for T in (1.0, 2.5):
        check(run(m_(), *a, T=T, ug=0.75, how=how), *reference(*a, T=T, ug=0.75), what=f"{size} {T}")


@pytest.mark.parametrize("how", ["step", "two calls"])
@pytest.mark.parametrize("size", [(6, 9, 8), (40, 1001, 300), (2, 40000, 1024)], ids=str)
def test_same_class_many_times(size, how):
    a = inputs(*size, seed=1, repeat=True)
    check(run(m_(), *a, how=how), *reference(*a), what=str(size))
    g = np.random.RandomState(0).standard_normal(a[0].shape).astype(np.float32)
    got, plain = run(m_(), *a, how=how, grad=g)["grad_x"], run(m_(), *a, how=how)["grad_x"]
    assert np.array_equal(got, g + plain)


@pytest.mark.parametrize("how", ["step", "two calls"])
@pytest.mark.parametrize("size", [(70, 999, 20), (300, 33000, 9), (3, 70001, 30), (258, 65541, 4)], ids=str)
def test_accumulates(size, how):
    a = inputs(*size, seed=2)
    g = np.random.RandomState(0).standard_normal(a[0].shape).astype(np.float32)
    got, plain = run(m_(), *a, how=how, grad=g)["grad_x"], run(m_(), *a, how=how)["grad_x"]
    assert np.array_equal(got, g + plain)


def test_same_bits_again():
    for size in ((70, 999, 20), (300, 33000, 9), (3, 70001, 30)):
        a = inputs(*size, seed=3)
        one, two = run(m_(), *a), run(m_(), *a)
        for k in one:
            assert np.array_equal(one[k], two[k]), (size, k)


@pytest.mark.parametrize("classes", [500, 40000])
def test_rows_left_out_may_hold_anything(classes):
    m = m_()
    x, ids, teacher = inputs(12, classes, 6, seed=4, left_out=0)
    ids[[1, 4, 7]] = -1
    teacher[9] = -np.inf
    want, bound = reference(x, ids, teacher)
    x[1], x[4], x[7], x[9] = np.nan, np.inf, 3e38, -np.inf
    teacher[1] = np.nan
    for how in ("step", "two calls"):
        check(run(m, x, ids, teacher, how=how), want, bound, how)
        got = run(m, x, ids, teacher, how=how, grad=np.full(x.shape, -0.0, np.float32))["grad_x"]
        assert (got[[1, 4, 7, 9]].view(np.uint32) == 0x80000000).all()


def test_no_row_left_and_no_rows():
    m = m_()
    x, ids, teacher = inputs(5, 300, 6, seed=5)
    for how in ("step", "two calls"):
        got = run(m, np.full_like(x, np.nan), np.full_like(ids, -1), teacher, how=how)
        assert got["loss"] == 0 and not got["row_lse"].any() and not got["grad_x"].any()
        assert run(m, x[:0], ids[:0], teacher[:0], how=how)["loss"] == 0


@pytest.mark.parametrize("low", [-np.inf, -3.4028234663852886e38])
@pytest.mark.parametrize("classes", [301, 40001])
def test_masked_logits(low, classes):
    """Logits at minus infinity, or the type's lowest value, have probability 0 and gradient 0."""
    x, ids, teacher = inputs(9, classes, 6, seed=6, left_out=0)
    r = np.random.RandomState(7)
    mask = r.uniform(size=x.shape) < 0.5
    mask[np.arange(9)[:, None], ids] = False
    x[mask] = low
    x[0] = low  # but for the entries
    x[0, ids[0]] = 1.5
    teacher[2, 1:] = -np.inf
    teacher[3, 2] = -3.4028234663852886e38
    for how in ("step", "two calls"):
        got = run(m_(), x, ids, teacher, how=how)
        check(got, *reference(x, ids, teacher), what=how)
        assert not got["grad_x"][mask].any()


@pytest.mark.parametrize("classes", [100, 40000])
def test_id_past_the_classes_shows(classes):
    for bad in (classes, 2147483647):
        x, ids, teacher = inputs(9, classes, 6, seed=8, left_out=0)
        ids[4, 3] = bad
        for how in ("step", "two calls"):
            got = run(m_(), x, ids, teacher, how=how)
            assert np.isnan(got["loss"]) and np.isnan(got["row_lse"][4]) and np.isnan(got["grad_x"][4]).all()
            assert np.isfinite(np.delete(got["row_lse"], 4)).all() and np.isfinite(np.delete(got["grad_x"], 4, 0)).all()


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_not_finite_shows(value):
    for classes in (100, 40000):
        x, ids, teacher = inputs(9, classes, 6, seed=9, left_out=0)
        x[4, classes - 1] = value
        got = run(m_(), x, ids, teacher)
        assert np.isnan(got["loss"]) and np.isnan(got["row_lse"][4]) and np.isnan(got["grad_x"][4]).all()
        assert np.isfinite(np.delete(got["grad_x"], 4, 0)).all()


def test_extreme_scales():
    x, ids, teacher = inputs(9, 777, 6, seed=10)
    for s, T in ((1e4, 1.0), (1e30, 1e6), (1e-30, 1e-6), (100.0, 0.01)):
        xs = (x * np.float32(s)).astype(np.float32)
        check(run(m_(), xs, ids, teacher, T=T), *reference(xs, ids, teacher, T=float(np.float32(T))), what=f"{s} {T}")


def test_gradient_against_differences():
    """The loss's third derivative along d is that of a log-sum-exp, at most 2 (max |d| / T)^3 T^2 a row; the loss
    in fp32 is off by 2^-22 of the terms it sums."""
    x, ids, teacher = inputs(8, 30, 4, seed=11)
    T, h = 1.5, 2.0 ** -6
    d = np.random.RandomState(1).standard_normal(x.shape).astype(np.float32)
    g = run(m_(), x, ids, teacher, T=T)["grad_x"].astype(np.float64)
    a, b = ((x + np.float32(s) * d).astype(np.float32) for s in (h, -h))
    quotient = (float(run(m_(), a, ids, teacher, T=T)["loss"]) - float(run(m_(), b, ids, teacher, T=T)["loss"])) / (2 * h)
    cubed = ((np.abs(d).max(1).astype(np.float64) / T) ** 3).mean() * T * T
    tol = cubed * h * h / 3 + 2.0 ** -22 * 10 * T * T / h
    assert abs(quotient - (g * d).sum()) <= tol and tol < abs(quotient), (quotient, (g * d).sum(), tol)


def test_unaligned_memory():
    m = m_()
    for size in ((5, 1001, 7), (2, 40001, 9)):
        x, ids, teacher = inputs(*size, seed=12)
        want = run(m, x, ids, teacher)
        hold = [(m.IndexTensor if a.dtype == np.int32 else m.Tensor).from_numpy(np.concatenate([[0], a.reshape(-1)]).astype(a.dtype))
                for a in (x, ids, teacher)]
        gx = m.Tensor(x.size + 2)
        loss = m.Tensor(1)
        m.distill_step(loss, m.Tensor.over(gx.ptr + 4, x.shape), m.Tensor.over(hold[0].ptr + 4, x.shape),
                       m.IndexTensor.over(hold[1].ptr + 4, ids.shape), m.Tensor.over(hold[2].ptr + 4, teacher.shape),
                       m.Tensor.from_numpy(np.float32([1])), accumulate=False)
        got = gx.to_numpy()
        assert np.array_equal(got[1:-1].reshape(x.shape), want["grad_x"]) and got[0] == 0 and got[-1] == 0
