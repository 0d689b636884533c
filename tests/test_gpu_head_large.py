"""The vocabulary head's cross entropy at sizes that are cut into several rounds: rows of a forward, elements a thread,
summation lengths."""
import numpy as np
import pytest

from test_gpu_head import check, inputs, m_, reference, run
from util import TEST_ASYNC

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def give_the_scratch_back():
    """These sizes grow the library's scratch to tens of GB, which it keeps until it is shut down."""
    yield
    m = m_()
    m._lib.call("mh_shutdown")
    m.init(0, asynchronous=TEST_ASYNC)


def forward(m, x, w, labels):
    rows = x.shape[0]
    loss, lse, rl = m.Tensor(1), m.Tensor(rows), m.Tensor(rows)
    m.linear_cross_entropy_forward(loss, lse, m.Tensor.from_numpy(x), m.Tensor.from_numpy(w), m.IndexTensor.from_numpy(labels), row_loss=rl)
    return {"loss": loss.to_numpy()[0], "row_lse": lse.to_numpy(), "row_loss": rl.to_numpy()}


def test_forward_cut_by_its_statistics():
    """2^24 classes: 2048 rows at once. Rows of eight kinds, whose results are those of one row of each, bit for bit; those
    against 64 bits."""
    m = m_()
    rows, classes = 2100, (1 << 24) - 5
    r = np.random.RandomState(61)
    kinds = r.standard_normal((8, 2)).astype(np.float32)
    w = r.standard_normal((classes, 2)).astype(np.float32)
    some = r.randint(0, classes, 8).astype(np.int32)
    which = r.randint(0, 8, rows)
    labels = some[which]
    labels[::11] = -1
    print("\n[head] forward in two cuts", flush=True)
    got = forward(m, kinds[which], w, labels)
    keep = labels >= 0
    one, bound = [], []
    for k in range(8):
        want, b = reference(kinds[k:k + 1], w, some[k:k + 1])
        one.append(want)
        bound.append(b)
    for name in ("row_lse", "row_loss"):
        want = np.array([o[name][0] for o in one])[which] * keep
        tol = np.array([b[name][0] for b in bound])[which] * keep
        assert (np.abs(got[name] - want) <= tol).all(), name
        assert not got[name][~keep].any()
        for k in range(8):
            same = got[name][keep & (which == k)]
            assert (same == same[0]).all(), (name, k)
    loss = (np.array([o["row_loss"][0] for o in one])[which] * keep).sum() / keep.sum()
    assert abs(got["loss"] - loss) <= max(b["row_loss"][0] for b in bound)


def test_gradient_sums_over_millions_of_classes():
    """2^25 classes: grad_x's sums run over at most 65536 of them at a time. All terms are positive, so that an adder's
    drift, 4e-11 of the sum an element, shows: 2.6e-6 then, 2.1e-5 over the 2^19 of one split in 64. The halves'
    roundings (2^-22 and, of an element of G near 2^-25, 2^-15 of itself) are as good as random over 2^25 terms."""
    m = m_()
    rows, dim, classes = 3, 4, 1 << 25
    tw = m.Tensor(classes, dim)
    m._lib.call("mh_rand_uniform", tw.ptr, classes * dim, 62, 0.5, 1.5)
    w = tw.to_numpy()
    labels = np.array([5, 6, 7], np.int32)
    zero = np.zeros((8, dim), np.float32)  # the labels' classes: -w_label adds nothing
    m._lib.call("mh_memcpy_h2d", tw.ptr, zero.ctypes.data, zero.nbytes)
    w[:8] = 0.0
    x = (0.01 * np.random.RandomState(63).standard_normal((rows, dim))).astype(np.float32)
    print("\n[head] 2^25 classes", flush=True)
    gx, loss = m.Tensor(rows, dim), m.Tensor(1)
    m.linear_cross_entropy_step(loss, gx, None, m.Tensor.from_numpy(x), tw, m.IndexTensor.from_numpy(labels),
                                m.Tensor.from_numpy(np.float32([rows])), accumulate=False)
    got = gx.to_numpy().astype(np.float64)
    want = np.zeros((rows, dim))
    total = np.zeros(rows)
    for v in range(0, classes, 1 << 21):
        part = w[v:v + (1 << 21)].astype(np.float64)
        e = np.exp(part @ x.T.astype(np.float64))
        total += e.sum(0)
        want += e.T @ part
    want /= total[:, None]
    off = np.abs(got / want - 1)
    print("[head] off by", off.max(), flush=True)
    assert off.max() <= 5e-6


def test_forward_of_more_rows_than_at_once():
    """33000 rows: 32768 and the rest, through the same statistics and targets."""
    x, w, labels = inputs(33000, 8, 70, seed=64)
    want, bound = reference(x, w, labels)
    check(forward(m_(), x, w, labels), want, bound, "rows")
    for how in ("step", "two calls"):
        check(run(m_(), x, w, labels, how=how), want, bound, how)


@pytest.mark.parametrize("place", ["first", "last"])
def test_a_wide_w_whose_largest_is_at_an_end(place):
    """10M elements of w: eight loads a thread and the rest. The power of two follows the largest wherever it lies: with
    another one's products would overflow their halves."""
    rows, dim, classes = 70, 100, 104003
    x, w, labels = inputs(rows, dim, classes, seed=65)
    at = (0, 3) if place == "first" else (classes - 1, dim - 1)
    w[at] = 3000.0
    x[:, at[1]] *= np.float32(1e-3)  # keeps the logits' size
    want, bound = reference(x, w, labels)
    floor = 2.0 ** -39 * (3000.0 * np.abs(x).sum(1) + np.abs(x).max(1) * np.abs(w).sum(1).max())
    bound["row_lse"], bound["row_loss"] = bound["row_lse"] + floor, bound["row_loss"] + 2 * floor
    bound["loss"] += 2 * floor.max()
    bound["grad_x"] = bound["grad_x"] + (2.0 ** -39 * 3000.0 * 2 + 3 * floor[:, None] * np.abs(w).max(0)[None]) / rows
    bound["grad_w"] = bound["grad_w"] + 3 * floor.max() * np.abs(x).max() / rows
    for how in ("step", "two calls"):
        check(run(m_(), x, w, labels, how=how), want, bound, f"{place} {how}")


def test_a_w_of_more_than_2_31_elements():
    """[131072, 16400] = 8.6 GB: offsets that pass 32 bits, in elements and in bytes. w is 0 but for classes at the ends
    and on either side of 2^31 and 2^32 bytes and 2^31 elements, so that the rest of the logits are 0."""
    m = m_()
    rows, dim, classes = 130, 16400, 131072
    assert rows > 128 and dim * classes > 1 << 31
    r = np.random.RandomState(66)
    some = sorted({0, 1, classes - 1} | {b // dim + d for b in (1 << 29, 1 << 30, (1 << 31) - dim) for d in (0, 1) if b // dim + d < classes})
    ws = (r.standard_normal((len(some), dim)) * 2 / np.sqrt(dim)).astype(np.float32)
    x = r.standard_normal((rows, dim)).astype(np.float32)
    labels = np.array(some, np.int32)[r.randint(0, len(some), rows)]
    labels[3] = -1
    w, gw, gx, loss, lse = m.Tensor(classes, dim), m.Tensor(classes, dim), m.Tensor(rows, dim), m.Tensor(1), m.Tensor(rows)
    for v, row in zip(some, ws):
        m._lib.call("mh_memcpy_h2d", w.ptr + 4 * v * dim, row.ctypes.data, 4 * dim)
    print("\n[head] 2^31 elements", flush=True)
    m.linear_cross_entropy_step(loss, gx, gw, m.Tensor.from_numpy(x), w, m.IndexTensor.from_numpy(labels),
                                m.Tensor.from_numpy(np.float32([1])), row_lse=lse, accumulate=False)
    keep = labels >= 0
    n = int(keep.sum())
    xd, wd = np.where(keep[:, None], x, 0.0).astype(np.float64), ws.astype(np.float64)
    z = xd @ wd.T
    total = np.exp(z).sum(1) + (classes - len(some))
    want = np.where(keep, np.log(total), 0.0)
    p = np.exp(z) / total[:, None]
    hit = labels[:, None] == np.array(some)[None]
    g = (p - hit) * keep[:, None] / n
    # bounds of test_gpu_head.py: a product of 16400 terms, the sums of 131072 exponentials
    U = 2.0 ** -24
    bz = (np.abs(xd) @ np.abs(wd).T) * (2.0 ** -21 + (3 * dim / 16 + 8) * 2 * U)
    bl = (p * bz).sum(1) + (128 + classes / 512 + 40) * U + 4 * U * want
    assert (np.abs(lse.to_numpy() - want)[keep] <= bl[keep]).all()
    row = want - (z * hit).sum(1)
    assert abs(loss.to_numpy()[0] - row[keep].mean()) <= (bl + bz.max(1) + 8 * U * (want + np.abs(z).max(1))).max()
    dg = (p * (bz + bl[:, None] + 2.0 ** -20) + 2.0 ** -22 * np.abs(g) * n + 2.0 ** -40) / n
    off = np.abs(gx.to_numpy() - g @ wd)
    assert (off <= dg @ np.abs(wd) + (np.abs(g) @ np.abs(wd)) * (2.0 ** -21 + 3 * 65536 / 16 * 2 * U) + 1e-12).all()
    part = np.empty((len(some), dim), np.float32)
    for i, v in enumerate(some):
        m._lib.call("mh_memcpy_d2h", part[i].ctypes.data, gw.ptr + 4 * v * dim, 4 * dim)
    off = np.abs(part - g.T @ xd)
    assert (off <= dg.T @ np.abs(xd) + (np.abs(g).T @ np.abs(xd)) * (2.0 ** -21 + 200 * U) + 1e-12).all()
    other = np.empty(dim, np.float32)  # a class of zeros: its probability times x
    m._lib.call("mh_memcpy_d2h", other.ctypes.data, gw.ptr + 4 * (classes - 2) * dim, 4 * dim)
    q = keep / total / n
    tol = (q * (bl + 2.0 ** -20) + 2.0 ** -40 / n) @ np.abs(xd) + (q @ np.abs(xd)) * (2.0 ** -21 + 200 * U)
    assert (np.abs(other - q @ xd) <= tol).all()
