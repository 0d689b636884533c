"""The vocabulary head's cross entropy (linear_cross_entropy_*) against the formulas in 64 bits.

Tolerances, from the arithmetic: an operand is held with 22 bits (2^-23 of itself off, and the product of
two remainders, below 2^-22, is dropped), so a product is off by 2^-21 of |x w| at most. A sum over K
elements takes 3 K / 16 additions into an fp32 accumulator, each off by at most 2^-23 of the sum so far
(a truncating adder; a rounding one has half). From these: Z, the bound of a logit; then a log-sum-exp is
off by Z, the sums' roundings and the log's; an element of G by p (Z + L + 2^-21) and 2^-22 of itself or
2^-40; a gradient by the sum of |dG| |operand| and its own product's bound."""
import numpy as np
import pytest

from util import GpuEngine

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def m_():
    return GpuEngine().m


def reference(x, w, labels, ug=1.0):
    """loss, row_loss, row_lse, grad_x, grad_w and the bounds of their errors."""
    labels = labels.astype(np.int64)
    keep = labels >= 0
    x, w = np.where(keep[:, None], x, 0.0).astype(np.float64), w.astype(np.float64)
    n = max(1, int(keep.sum()))
    rows, dim = x.shape
    classes = w.shape[0]
    z = x @ w.T
    top = z.max(1, keepdims=True)
    lse = top[:, 0] + np.log(np.exp(z - top).sum(1))
    at = np.arange(rows), np.maximum(labels, 0)
    picked = z[at]
    row = np.where(keep, lse - picked, 0.0)
    p = np.exp(z - lse[:, None])
    g = p.copy()
    g[at] -= 1.0
    g *= keep[:, None]
    c = ug / n

    def product(k):
        return 2.0 ** -21 + (3 * k / 16 + 8) * 2 * U

    ax, aw, ag = np.abs(x), np.abs(w), np.abs(g)
    bz = (ax @ aw.T) * product(dim)
    # 64 or 128 terms a lane, then the groups' statistics
    bl = bz.max(1) + (128 + classes / 512 + 40) * U + 4 * U * np.abs(lse)
    brow = bl + bz[at] + 4 * U * (np.abs(lse) + np.abs(picked))
    dg = p * (bz + bl[:, None] + 2.0 ** -21 + 8 * U * (np.abs(z) + np.abs(lse)[:, None])) + 2.0 ** -22 * ag + 2.0 ** -40
    dg *= keep[:, None]
    bgx = abs(c) * (dg @ aw + (ag @ aw) * product(classes + 256))
    bgw = abs(c) * (dg.T @ ax + (ag.T @ ax) * product(rows + 256))
    out = {"loss": row.sum() / n, "row_loss": row, "row_lse": np.where(keep, lse, 0.0), "grad_x": c * (g @ w), "grad_w": c * (g.T @ x)}
    bound = {"loss": (brow * keep).sum() / n + 4 * U * abs(out["loss"]), "row_loss": brow * keep, "row_lse": bl * keep,
             "grad_x": bgx + 4 * U * np.abs(out["grad_x"]), "grad_w": bgw + 4 * U * np.abs(out["grad_w"])}
    return out, bound


def inputs(rows, dim, classes, seed, left_out=0.1, std=2.0):
    r = np.random.RandomState(seed)
    x = r.standard_normal((rows, dim)).astype(np.float32)
    w = (r.standard_normal((classes, dim)) * std / np.sqrt(dim)).astype(np.float32)
    labels = r.randint(0, classes, rows).astype(np.int32)
    labels[r.uniform(size=rows) < left_out] = -100
    return x, w, labels


def run(m, x, w, labels, ug=1.0, how="step", grads=None):
    """The results by name. `grads`: (grad_x, grad_w) that the gradients are added to."""
    rows, dim = x.shape
    classes = w.shape[0]
    tx, tw, tl, tu = m.Tensor.from_numpy(x), m.Tensor.from_numpy(w), m.IndexTensor.from_numpy(labels), m.Tensor.from_numpy(np.float32([ug]))
    loss, lse, rl = m.Tensor(1), m.Tensor(rows), m.Tensor(rows)
    add = grads is not None
    fill = np.full  # what accumulate=False has to write over
    gx = m.Tensor.from_numpy(grads[0] if add else fill((rows, dim), 7.0, np.float32))
    gw = m.Tensor.from_numpy(grads[1] if add else fill((classes, dim), 7.0, np.float32))
    if how == "step":
        m.linear_cross_entropy_step(loss, gx, gw, tx, tw, tl, tu, row_lse=lse, accumulate=add)
    else:
        m.linear_cross_entropy_forward(loss, lse, tx, tw, tl, row_loss=rl)
        m.linear_cross_entropy_backward(gx, gw, tx, tw, tl, lse, tu, accumulate=add)
    out = {"loss": loss.to_numpy()[0], "row_lse": lse.to_numpy(), "grad_x": gx.to_numpy(), "grad_w": gw.to_numpy()}
    if how != "step":
        out["row_loss"] = rl.to_numpy()
    return out


def check(got, want, bound, what=""):
    for k, v in got.items():
        off = np.abs(v.astype(np.float64) - want[k])
        assert np.isfinite(v).all(), f"{what} {k}: not finite"
        over = off > bound[k] + 1e-42
        assert not over.any(), f"{what} {k}: {over.sum()} of {over.size} beyond the bound, worst {off.max():.3g} of {np.max(bound[k]):.3g}"
        # the roundings are as good as random: their sum is far below the bound of the worst case
        norm = np.linalg.norm(want[k])
        if norm > 0 and k.startswith("grad"):
            assert np.linalg.norm(off) <= 1e-5 * norm, f"{what} {k}: {np.linalg.norm(off) / norm:.3g} off in the norm"


SIZES = [(1, 1, 1), (1, 1, 2), (2, 3, 5), (1, 70, 300), (16, 64, 1000), (31, 33, 63), (33, 100, 257), (64, 128, 256),
         (257, 31, 2049), (300, 129, 5003), (130, 513, 999), (1024, 40, 130), (255, 16, 256), (256, 32, 8191)]


@pytest.mark.parametrize("how", ["step", "two calls"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, how):
    print(f"\n[head] {size} {how}", flush=True)
    x, w, labels = inputs(*size, seed=sum(size))
    want, bound = reference(x, w, labels, ug=0.75)
    check(run(m_(), x, w, labels, ug=0.75, how=how), want, bound, str(size))


def test_larger_tiles_and_splits():
    """Products of whole 256 x 256 tiles, and gradients whose long axis is split."""
    m = m_()
    for size in ((4096, 96, 5000), (2048, 300, 9001), (300, 2500, 4000)):
        print(f"\n[head] {size}", flush=True)
        x, w, labels = inputs(*size, seed=3)
        want, bound = reference(x, w, labels)
        check(run(m, x, w, labels), want, bound, str(size))


@pytest.mark.parametrize("size", [(1, 513, 9001), (16, 4097, 1031), (32, 1024, 4100), (33, 700, 6007), (64, 2050, 2049), (65, 1030, 4111), (128, 512, 8200), (9, 257, 16390), (9, 48, 100003)], ids=str)
def test_few_rows_against_a_large_head(size):
    """Up to 64 rows, 128 forward: w read as it lies, three bf16 an element, whose products are off by 2^-22 at most."""
    m = m_()
    x, w, labels = inputs(*size, seed=21)
    labels[0] = 3
    want, bound = reference(x, w, labels)
    for how in ("step", "two calls"):
        check(run(m, x, w, labels, how=how), want, bound, how)
    r = np.random.RandomState(1)
    g0 = r.standard_normal(x.shape).astype(np.float32), r.standard_normal(w.shape).astype(np.float32)
    plain, got = run(m, x, w, labels), run(m, x, w, labels, grads=g0)
    assert np.array_equal(got["grad_w"], g0[1] + plain["grad_w"]) and np.array_equal(got["grad_x"], g0[0] + plain["grad_x"])
    if size[0] > 4:  # rows left out, classes that do not exist, infinities
        labels[1], x[1] = -5, np.nan
        labels[2] = size[2]
        got = run(m, x, w, labels)
        assert np.isnan(got["row_lse"][2]) and got["row_lse"][1] == 0 and not got["grad_x"][1].any()
        assert np.isfinite(np.delete(got["grad_x"], 2, 0)).all() and np.isnan(got["grad_x"][2]).all()
        labels[2] = 0
        w[5, 7] = np.inf
        assert np.isnan(run(m, x, w, labels)["loss"])


def test_rows_in_chunks():
    """2^20 classes: the logits of 512 rows at a time, the last chunk shorter, grad_w over both."""
    rows, classes = 600, 1 << 20
    x, w, labels = inputs(rows, 4, classes, seed=5)
    print("\n[head] chunks", flush=True)
    got = run(m_(), x, w, labels)
    two = run(m_(), x, w, labels, how="two calls")
    for k in got:
        assert np.array_equal(got[k], two[k]), k
    # every row's log-sum-exp and loss, 40 rows at a time; the gradients of some rows and some classes, with
    # reference()'s bounds, which grow with a logit's size (four elements make logits beyond +-30, whose fp32
    # step alone is 2^-20 of e^z)
    keep, n = labels >= 0, int((labels >= 0).sum())
    some = np.concatenate([np.arange(3), np.arange(508, 516), np.arange(597, 600)])
    part = np.sort(np.concatenate([np.random.RandomState(1).choice(classes, 300, replace=False), labels[keep][:200]]))
    xd, wd = np.where(keep[:, None], x, 0.0).astype(np.float64), w.astype(np.float64)
    lse, loss = np.zeros(rows), 0.0
    for r in range(0, rows, 40):
        z = xd[r:r + 40] @ wd.T
        top = z.max(1, keepdims=True)
        picked = z[np.arange(len(z)), np.maximum(labels[r:r + 40], 0)]
        np.subtract(z, top, out=z)
        lse[r:r + 40] = top[:, 0] + np.log(np.exp(z, out=z).sum(1))
        loss += ((lse[r:r + 40] - picked) * keep[r:r + 40]).sum() / n
    one, bound = reference(x[some], w, labels[some])
    share = int(keep[some].sum()) / n
    check({"row_lse": got["row_lse"][some], "grad_x": got["grad_x"][some]}, {"row_lse": one["row_lse"], "grad_x": one["grad_x"] * share},
          {"row_lse": bound["row_lse"], "grad_x": bound["grad_x"] * share}, "some rows")
    assert np.allclose(got["row_lse"][keep], lse[keep], rtol=2e-6) and abs(got["loss"] - loss) <= 2e-6 * loss
    z = xd @ wd[part].T
    p = np.exp(z - lse[:, None])
    g = p - (part[None, :] == labels[:, None])
    g *= keep[:, None]
    bz = (np.abs(xd) @ np.abs(wd[part]).T) * 2.0 ** -20
    dg = p * (bz + 2.0 ** -14 + 8 * U * (np.abs(z) + lse[:, None])) + 2.0 ** -22 * np.abs(g) + 2.0 ** -40
    # 2^-14: the log-sum-exp's own bound there is (128 + 2^20 / 512) U and the largest logit's
    bw = ((dg * keep[:, None]).T @ np.abs(xd) + (np.abs(g).T @ np.abs(xd)) * (2.0 ** -21 + 150 * U)) / n
    check({"grad_w": got["grad_w"][part]}, {"grad_w": g.T @ xd / n}, {"grad_w": bw}, "some classes")


def test_accumulates():
    m = m_()
    x, w, labels = inputs(70, 50, 600, seed=9)
    r = np.random.RandomState(1)
    g0 = r.standard_normal((70, 50)).astype(np.float32), r.standard_normal((600, 50)).astype(np.float32)
    plain = run(m, x, w, labels)
    for how in ("step", "two calls"):
        got = run(m, x, w, labels, how=how, grads=g0)
        assert np.array_equal(got["grad_x"], g0[0] + plain["grad_x"])
        assert np.array_equal(got["grad_w"], g0[1] + plain["grad_w"])


def test_same_bits_again_and_in_both_forms():
    m = m_()
    x, w, labels = inputs(300, 200, 3001, seed=10)
    one, two, three = run(m, x, w, labels), run(m, x, w, labels), run(m, x, w, labels, how="two calls")
    for k in one:
        assert np.array_equal(one[k], two[k]) and np.array_equal(one[k], three[k]), k


def test_rows_left_out_may_hold_anything():
    m = m_()
    x, w, labels = inputs(90, 65, 500, seed=11, left_out=0.3)
    want, bound = reference(x, w, labels)
    out = np.flatnonzero(labels < 0)
    bad = x.copy()
    bad[out[0]], bad[out[1]], bad[out[2]], bad[out[3:]] = np.nan, np.inf, 3e38, -3.4028234663852886e38
    labels[out[0]] = -1
    labels[out[1]] = -2147483648
    check(run(m, bad, w, labels), want, bound, "left out")
    g0 = np.full((90, 65), -0.0, np.float32), np.zeros((500, 65), np.float32)
    got = run(m, bad, w, labels, grads=g0)
    assert (got["grad_x"][out].view(np.uint32) == 0x80000000).all()  # left as they were


def test_no_row_kept():
    m = m_()
    x, w, labels = inputs(40, 20, 100, seed=12)
    labels[:] = -1
    x[:] = np.nan
    for how in ("step", "two calls"):
        got = run(m, x, w, labels, how=how)
        assert got["loss"] == 0 and not got["row_lse"].any() and not got["grad_x"].any() and not got["grad_w"].any()


def test_no_rows():
    m = m_()
    x, w, labels = np.zeros((0, 20), np.float32), np.ones((30, 20), np.float32), np.zeros(0, np.int32)
    for how in ("step", "two calls"):
        got = run(m, x, w, labels, how=how)
        assert got["loss"] == 0 and not got["grad_w"].any()
        assert (run(m, x, w, labels, how=how, grads=(x, w))["grad_w"] == 1).all()


def test_label_past_the_classes_shows():
    m = m_()
    for label in (100, 2147483647):
        x, w, labels = inputs(40, 20, 100, seed=13)
        labels[:] = np.arange(40)
        labels[7] = label
        got = run(m, x, w, labels)
        assert np.isnan(got["loss"]) and np.isnan(got["row_lse"][7]) and np.isfinite(np.delete(got["row_lse"], 7)).all()
        assert np.isnan(got["grad_x"][7]).all() and np.isfinite(np.delete(got["grad_x"], 7, 0)).all()
        assert np.isnan(got["grad_w"]).all()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_not_finite_shows(value):
    m = m_()
    x, w, labels = inputs(40, 20, 100, seed=14, left_out=0)
    x[3, 5] = value
    got = run(m, x, w, labels)
    assert np.isnan(got["loss"]) and np.isnan(got["row_lse"][3]) and np.isfinite(np.delete(got["row_lse"], 3)).all()
    x, w, labels = inputs(40, 20, 100, seed=14, left_out=0)
    w[99, 19] = value
    assert np.isnan(run(m, x, w, labels)["loss"])


@pytest.mark.parametrize("sx, sw", [(1e4, 1e-6), (1e-20, 1e20), (1e-30, 1e15), (1e18, 1e-18), (0.0, 1.0), (1.0, 0.0), (1.0, 40.0)])
def test_scales(sx, sw):
    """Operands of any scale: the powers of two follow the largest element. The last: logits to +-300."""
    m = m_()
    x, w, labels = inputs(65, 40, 333, seed=15)
    x, w = (x * np.float32(sx)).astype(np.float32), (w * np.float32(sw)).astype(np.float32)
    want, bound = reference(x, w, labels)
    got = run(m, x, w, labels)
    for k in got:
        off = np.abs(got[k].astype(np.float64) - want[k])
        # results below the least normal number round to a step of 2^-149
        assert (off <= bound[k] + 2.0 ** -148).all(), (k, off.max())


def test_one_gradient_only():
    m = m_()
    x, w, labels = inputs(70, 50, 600, seed=16)
    both = run(m, x, w, labels)
    tx, tw, tl, tu = m.Tensor.from_numpy(x), m.Tensor.from_numpy(w), m.IndexTensor.from_numpy(labels), m.Tensor.from_numpy(np.float32([1]))
    loss, gx, gw = m.Tensor(1), m.Tensor(70, 50), m.Tensor(600, 50)
    m.linear_cross_entropy_step(loss, gx, None, tx, tw, tl, tu)
    assert np.array_equal(gx.to_numpy(), both["grad_x"])
    m.linear_cross_entropy_step(loss, None, gw, tx, tw, tl, tu)
    assert np.array_equal(gw.to_numpy(), both["grad_w"])
    m.linear_cross_entropy_step(loss, None, None, tx, tw, tl, tu)
    assert loss.to_numpy()[0] == both["loss"]


def test_gradients_against_differences():
    """<grad, d> against (loss(+h d) - loss(-h d)) / 2 h. The loss is off by up to 2^-22 of its size, so the
    quotient by 2^-22 loss / h; the third derivative of a row's log-sum-exp along d is at most 2 (max |z'|)^3,
    the loss is the rows' mean, and the quotient's error a sixth of its third derivative times h^2."""
    m = m_()
    x, w, labels = inputs(24, 12, 50, seed=17)
    g = run(m, x, w, labels)
    r = np.random.RandomState(2)
    for which in ("x", "w"):
        a = x if which == "x" else w
        d = r.standard_normal(a.shape).astype(np.float32)
        h = 2.0 ** -6
        loss, slope = [], 0.0
        for s in (h, -h):
            a2 = (a + np.float32(s) * d).astype(np.float32)
            xx, ww = (a2, w) if which == "x" else (x, a2)
            loss.append(float(run(m, xx, ww, labels)["loss"]))
        row = np.abs(d @ w.T if which == "x" else x @ d.T).max(1).astype(np.float64)
        slope, cubed = row.max(), (row ** 3).mean()
        quotient, inner = (loss[0] - loss[1]) / (2 * h), float((g["grad_" + which].astype(np.float64) * d).sum())
        tol = 2.0 ** -22 * loss[0] / h + cubed * h * h / 3 + 2.0 ** -23 * np.abs(a).max() * slope / h
        assert abs(quotient - inner) <= tol, (which, quotient, inner, tol)
        assert tol < abs(inner) or abs(inner) < 0.05


def test_memory_of_another_allocator():
    m = m_()
    x, w, labels = inputs(70, 51, 601, seed=18)
    want = run(m, x, w, labels)
    # odd addresses: views that start one element into an allocation
    hold = [(m.IndexTensor if a.dtype == np.int32 else m.Tensor).from_numpy(np.concatenate([[0], a.reshape(-1)]).astype(a.dtype)) for a in (x, w, labels)]
    gx, gw = m.Tensor(x.size + 2), m.Tensor(w.size + 2)
    tx, tw = (m.Tensor.over(t.ptr + 4, a.shape, t) for t, a in zip(hold, (x, w)))
    tl = m.IndexTensor.over(hold[2].ptr + 4, labels.shape, hold[2])
    loss, tu = m.Tensor(1), m.Tensor.from_numpy(np.float32([1]))
    m.linear_cross_entropy_step(loss, m.Tensor.over(gx.ptr + 4, x.shape), m.Tensor.over(gw.ptr + 4, w.shape),
                                tx, tw, tl, tu)
    for name, t, shape in (("grad_x", gx.to_numpy(), x.shape), ("grad_w", gw.to_numpy(), w.shape)):
        assert np.array_equal(t[1:-1].reshape(shape), want[name]) and t[0] == 0 and t[-1] == 0
