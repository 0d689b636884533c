"""Distillation over more rows than the entries' kernel takes at once, so that a wavefront goes round with the same hash
table, and over tensors of more than 2^31 elements. Bounds are those of test_gpu_distill.py; a row of up to 1024 classes is
summed by one wavefront, 16 elements a lane, of up to 8192 by four and of up to 16384 by eight, 32 a lane, so its bound
has classes / 64, / 256 and / 512 in the place of classes / 1024."""
import numpy as np
import pytest

from test_gpu_distill import NONE, U, check, inputs, m_, reference, run

pytestmark = pytest.mark.gpu


def lanes(classes, k):
    return 64 if classes <= 1024 and k <= 128 else 256 if classes <= 8192 else 512 if classes <= 16384 else 1024


def bounded(x, ids, teacher, **kw):
    """reference() with the elements that a thread sums."""
    want, bound = reference(x, ids, teacher, **kw)
    classes = x.shape[1]
    more = U * (classes / lanes(classes, ids.shape[1]) - classes / 1024)
    T, ug = kw.get("T", 1.0), kw.get("ug", 1.0)
    n = max(1, int((ids >= 0).any(1).sum()))
    bound["row_lse"] = bound["row_lse"] + more
    bound["loss"] += T * T * more
    y = np.where((ids >= 0).any(1)[:, None], x, 0.0).astype(np.float64) / T
    p = np.exp(y - y.max(1, keepdims=True))
    bound["grad_x"] = bound["grad_x"] + abs(ug) * T / n * more * p / p.sum(1, keepdims=True)
    return want, bound


@pytest.mark.parametrize("size", [(5000, 300, 9), (2500, 40, 600), (20000, 64, 16), (70000, 20, 3), (4500, 1000, 130), (1500, 9000, 1024)], ids=str)
def test_rounds_of_the_entries(size):
    """Classes that repeat, in every row: what a table held for the row before must be gone."""
    print(f"\n[distill] {size}", flush=True)
    a = inputs(*size, seed=81, repeat=True)
    rows, classes, k = size
    if classes > k:
        a[1][::2] = np.where(a[1][::2] >= 0, np.random.RandomState(82).randint(0, classes, a[1][::2].shape), a[1][::2])
    for how in ("step", "two calls"):
        check(run(m_(), *a, how=how), *bounded(*a), what=f"{size} {how}")


@pytest.mark.parametrize("classes", [700, 1024, 8192, 16384])
def test_sums_of_short_rows(classes):
    a = inputs(70, classes, 12, seed=83)
    for how in ("step", "two calls"):
        check(run(m_(), *a, how=how), *bounded(*a), what=f"{classes} {how}")


@pytest.mark.parametrize("rows, classes, k", [(16500, 131072, 7), (2200000, 1000, 2)])
def test_more_than_2_31_elements(rows, classes, k):
    """Offsets that pass 32 bits: the rows at both ends, and those on either side of 2^31 and 2^32 bytes and elements."""
    m = m_()
    r = np.random.RandomState(84)
    x, g = m.Tensor(rows, classes), m.Tensor(rows, classes)
    m._lib.call("mh_rand_normal", x.ptr, rows * classes, 85, 0.0, 2.0)
    m._lib.call("mh_fill", g.ptr, 7.0, rows * classes)
    ids = r.randint(0, classes, (rows, k)).astype(np.int32)
    ids[::13] = NONE
    teacher = r.standard_normal((rows, k)).astype(np.float32)
    ti, tt, one, loss, lse = m.IndexTensor.from_numpy(ids), m.Tensor.from_numpy(teacher), m.Tensor.from_numpy(np.float32([1])), m.Tensor(1), m.Tensor(rows)
    n = int((ids >= 0).any(1).sum())
    some = sorted({0, 1, rows - 2, rows - 1} | {b // classes + d for b in (1 << 29, 1 << 30, 1 << 31) for d in (-1, 0, 1) if b // classes + 1 < rows})
    xs = np.empty((len(some), classes), np.float32)

    def fetch(t, out):
        for i, row in enumerate(some):
            m._lib.call("mh_memcpy_d2h", out[i].ctypes.data, t.ptr + 4 * row * classes, 4 * classes)
        return out
    fetch(x, xs)
    want, bound = bounded(xs, ids[some], teacher[some])
    share = max(1, int((ids[some] >= 0).any(1).sum())) / n
    for how in ("step", "two calls"):
        print(f"\n[distill] {rows} {classes} {how}", flush=True)
        if how == "step":
            m.distill_step(loss, g, x, ti, tt, one, row_lse=lse, accumulate=False)
        else:
            m._lib.call("mh_fill", g.ptr, 7.0, rows * classes)
            m.distill_forward(loss, lse, x, ti, tt)
            m.distill_backward(g, x, ti, tt, lse, one, accumulate=False)
        got = {"grad_x": fetch(g, np.empty_like(xs)), "row_lse": lse.to_numpy()[some]}
        check(got, {"grad_x": want["grad_x"] * share, "row_lse": want["row_lse"]},
              {"grad_x": bound["grad_x"] * share, "row_lse": bound["row_lse"]}, how)
        assert np.isfinite(loss.to_numpy()).all()
