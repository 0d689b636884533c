"""The mixture-of-experts router (router_*) against the formulas in 64 bits.

Tolerances, U = 2^-24: an exponential is off by (|x - max| + 4) U of itself, a row's sum of E by 24 more (16 a
lane, the rest a tree), so a probability by R = (|x - max| + 40) U; sums over rows by rows / 1024 + 30 roundings,
counts are whole. A gradient p (A - sum A p) is off by p (|A| + sum |A| p) times twice R and 40 U."""
import numpy as np
import pytest

from util import GpuEngine

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def m_():
    return GpuEngine().m


def reference(x, k, keep=None, normalise=False, gw=None, ug=None):
    rows, experts = x.shape
    order = np.argsort(-(x + np.float32(0.0)), axis=1, kind="stable")[:, :k]
    kept = np.ones(rows, bool) if keep is None else keep != 0
    xd = np.where(kept[:, None], x, 0.0).astype(np.float64)
    n = max(1, int(kept.sum()))
    top = xd.max(1, keepdims=True)
    p = np.exp(xd - top)
    p /= p.sum(1, keepdims=True)
    counts = np.bincount(order[kept].reshape(-1), minlength=experts)
    r = np.arange(rows)[:, None]
    picked = p[r, order]
    mass = picked.sum(1, keepdims=True)
    weights = picked / mass if normalise else picked
    weights = np.where(kept[:, None], weights, 0.0)
    f = counts / (n * k)
    loss = experts * (f * (p * kept[:, None]).sum(0)).sum() / n
    s = 0.0 if ug is None else ug * experts / n
    grad = s * p * (f - (f * p).sum(1, keepdims=True))
    g = np.zeros((rows, experts))
    if gw is not None:
        gd = np.where(kept[:, None], gw, 0.0).astype(np.float64)
        if normalise:
            grad[r, order] += picked / mass * (gd - (gd * picked / mass).sum(1, keepdims=True))
        else:
            grad -= p * (gd * picked).sum(1, keepdims=True)
            grad[r, order] += picked * gd
        g[r, order] = np.abs(gd) / (mass if normalise else 1.0)  # the weights' own softmax: w is p / mass
    rel = (np.minimum(top - xd, 1e4) + 40) * U
    A = g + abs(s) * f
    bg = p * (A + (A * p).sum(1, keepdims=True) + (g * p).sum(1, keepdims=True) / mass) * (2 * rel + 40 * U)
    bw = weights * (rel[r, order] + rel[r, order].max(1, keepdims=True) + 80 * U)
    bl = experts * (f * (p * rel * kept[:, None]).sum(0)).sum() / n + (rows / 1024 + 40 + experts / 64) * U * loss
    out = {"weights": weights, "loss": loss, "grad_x": grad * kept[:, None]}
    bound = {"weights": bw, "loss": bl, "grad_x": bg * kept[:, None]}
    return out, bound, {"chosen": np.where(kept[:, None], order, -1), "counts": counts}


def run(m, x, k, keep=None, normalise=False, gw=None, ug=None, grad=None):
    rows, experts = x.shape
    tx = m.Tensor.from_numpy(x)
    tk = None if keep is None else m.IndexTensor.from_numpy(keep)
    weights, chosen, counts, loss = m.Tensor(rows, k), m.IndexTensor(rows, k), m.IndexTensor(experts), m.Tensor(1)
    m.router_forward(weights, chosen, counts, loss, tx, keep=tk, normalise=normalise)
    gx = m.Tensor.from_numpy(np.full(x.shape, 7.0, np.float32) if grad is None else grad)
    m.router_backward(gx, tx, chosen, counts, None if gw is None else m.Tensor.from_numpy(gw),
                      None if ug is None else m.Tensor.from_numpy(np.float32([ug])), keep=tk, normalise=normalise,
                      accumulate=grad is not None)
    return {"weights": weights.to_numpy(), "chosen": chosen.to_numpy(), "counts": counts.to_numpy(),
            "loss": loss.to_numpy()[0], "grad_x": gx.to_numpy()}


def check(got, want, bound, whole, what=""):
    for a, v in whole.items():
        assert np.array_equal(got[a], v), f"{what} {a}"
    for a, v in want.items():
        off = np.abs(got[a].astype(np.float64) - v)
        assert np.isfinite(got[a]).all(), f"{what} {a}: not finite"
        over = off > bound[a] + 1e-37
        assert not over.any(), f"{what} {a}: {over.sum()} of {over.size} beyond the bound, worst {off.max():.3g} of {np.max(bound[a]):.3g}"


def inputs(rows, experts, k, seed):
    r = np.random.RandomState(seed)
    x = (1.5 * r.standard_normal((rows, experts))).astype(np.float32)
    return x, (r.uniform(size=rows) > 0.1).astype(np.int32), r.standard_normal((rows, k)).astype(np.float32)


SIZES = [(1, 1, 1), (2, 2, 1), (7, 3, 3), (64, 8, 2), (65, 7, 2), (300, 9, 4), (1000, 16, 16), (33, 17, 5), (500, 32, 8),
         (700, 60, 6), (129, 64, 64), (300, 65, 8), (2000, 127, 4), (77, 128, 8), (90, 200, 16), (4099, 256, 8), (50, 257, 3),
         (40, 512, 64), (20, 1000, 10), (9, 1024, 64), (20000, 30, 2), (1, 1021, 7)]


@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, normalise):
    print(f"\n[router] {size} {normalise}", flush=True)
    x, keep, gw = inputs(*size, seed=sum(size))
    for kp in (None, keep):
        check(run(m_(), x, size[2], kp, normalise, gw, 0.3), *reference(x, size[2], kp, normalise, gw, 0.3), what=str(size))


@pytest.mark.parametrize("normalise", [False, True])
def test_one_gradient_alone(normalise):
    x, keep, gw = inputs(333, 40, 5, seed=1)
    for g, u in ((gw, None), (None, 0.7), (None, None)):
        check(run(m_(), x, 5, keep, normalise, g, u), *reference(x, 5, keep, normalise, g, u), what=f"{g is None} {u}")


@pytest.mark.parametrize("experts, k", [(8, 3), (64, 64), (100, 7), (1024, 20)])
def test_ties_go_to_the_lowest_index(experts, k):
    r = np.random.RandomState(2)
    x = r.randint(-2, 3, (200, experts)).astype(np.float32)
    x[r.uniform(size=x.shape) < 0.1] = -0.0
    x[3] = 0.5
    _, keep, gw = inputs(200, experts, k, seed=3)
    check(run(m_(), x, k, keep, True, gw, 1.0), *reference(x, k, keep, True, gw, 1.0), what="ties")


@pytest.mark.parametrize("low", [-np.inf, -3.4028234663852886e38])
def test_masked_experts(low):
    """Experts a mask leaves out come last, with weight and gradient 0."""
    x, keep, gw = inputs(100, 50, 6, seed=4)
    x[np.random.RandomState(5).uniform(size=x.shape) < 0.5] = low
    x[7] = low
    x[7, 20:23] = [1.0, 2.0, 0.5]  # fewer experts than k
    for normalise in (False, True):
        got = run(m_(), x, 6, keep, normalise, gw, 1.0)
        check(got, *reference(x, 6, keep, normalise, gw, 1.0), what=str(normalise))
        assert list(got["chosen"][7]) == [21, 20, 22, 0, 1, 2] or keep[7] == 0


def test_padding_rows_may_hold_anything():
    x, keep, gw = inputs(60, 33, 4, seed=6)
    keep[[3, 10, 20]] = 0
    want = reference(x, 4, keep, True, gw, 1.0)
    x[3], x[10], x[20], gw[3] = np.nan, np.inf, -np.inf, np.nan
    check(run(m_(), x, 4, keep, True, gw, 1.0), *want, what="padding")
    got = run(m_(), x, 4, keep, True, gw, 1.0, grad=np.full(x.shape, -0.0, np.float32))["grad_x"]
    assert (got[keep == 0].view(np.uint32) == 0x80000000).all()


def test_no_row_kept_and_no_rows():
    x, keep, gw = inputs(60, 33, 4, seed=7)
    got = run(m_(), x, 4, keep * 0, True, gw, 1.0)
    assert got["loss"] == 0 and not got["counts"].any() and (got["chosen"] == -1).all()
    assert not got["weights"].any() and not got["grad_x"].any()
    got = run(m_(), x[:0], 4, keep[:0], True, gw[:0], 1.0)
    assert got["loss"] == 0 and not got["counts"].any()


def test_accumulates():
    for size in ((70, 33, 4), (500, 256, 8), (129, 5, 2)):
        x, keep, gw = inputs(*size, seed=8)
        g = np.random.RandomState(0).standard_normal(x.shape).astype(np.float32)
        for normalise in (False, True):
            got = run(m_(), x, size[2], keep, normalise, gw, 1.0, grad=g)["grad_x"]
            assert np.array_equal(got, g + run(m_(), x, size[2], keep, normalise, gw, 1.0)["grad_x"])


def test_same_bits_again():
    x, keep, gw = inputs(5000, 100, 6, seed=9)
    one, two = (run(m_(), x, 6, keep, True, gw, 1.0) for _ in range(2))
    for a in one:
        assert np.array_equal(one[a], two[a]), a


def test_nan_comes_last():
    x, keep, gw = inputs(20, 12, 12, seed=10)
    x[5, 3] = np.nan
    got = run(m_(), x, 12)
    assert got["chosen"][5, 11] == 3 and sorted(got["chosen"][5]) == list(range(12))
    assert np.isnan(got["weights"][5]).all() and np.isfinite(np.delete(got["weights"], 5, 0)).all() and np.isnan(got["loss"])


def test_gradient_against_differences():
    """Away from ties the choice stays as it is over a small step, so the loss and weights are smooth: third
    derivatives along d of p, and of a quotient of sums of p, stay below 40 max |d|^3."""
    x, keep, gw = inputs(30, 10, 3, seed=11)
    d = np.random.RandomState(1).standard_normal(x.shape).astype(np.float32)
    h = 2.0 ** -8
    top = -np.sort(-x, 1)
    sure = (top[:, 2] - top[:, 3]) > 4 * h * np.abs(d).max()
    keep = (keep * sure).astype(np.int32)
    for normalise in (False, True):
        g = run(m_(), x, 3, keep, normalise, gw, 0.8)["grad_x"].astype(np.float64)
        val = []
        for s in (h, -h):
            y = (x + np.float32(s) * d).astype(np.float32)
            r = run(m_(), y, 3, keep, normalise)
            order = np.argsort(r["chosen"], 1), np.argsort(run(m_(), x, 3, keep, normalise)["chosen"], 1)
            # a pair inside the chosen may change places; match the weights by expert
            w = np.take_along_axis(r["weights"], order[0], 1)
            gws = np.take_along_axis(gw, order[1], 1)
            val.append(0.8 * float(r["loss"]) + float((w.astype(np.float64) * gws * keep[:, None]).sum()))
        quotient = (val[0] - val[1]) / (2 * h)
        third = 40 * (np.abs(d).max(1).astype(np.float64) ** 3 * (np.abs(gw).max(1) + 0.8)).sum() / 6
        assert abs(quotient - (g * d).sum()) <= third * h * h + 2.0 ** -21 * np.abs(gw).sum() / h, normalise


def test_unaligned_memory():
    m = m_()
    x, keep, gw = inputs(50, 37, 5, seed=12)
    want = run(m, x, 5, keep, True, gw, 1.0)
    tx = m.Tensor.from_numpy(np.concatenate([[0], x.reshape(-1)]).astype(np.float32))
    gx = m.Tensor(x.size + 2)
    X = m.Tensor.over(tx.ptr + 4, x.shape, tx)
    K = m.IndexTensor.from_numpy(keep)
    weights, chosen, counts, loss = m.Tensor(50, 5), m.IndexTensor(50, 5), m.IndexTensor(37), m.Tensor(1)
    m.router_forward(weights, chosen, counts, loss, X, keep=K, normalise=True)
    m.router_backward(m.Tensor.over(gx.ptr + 4, x.shape), X, chosen, counts, m.Tensor.from_numpy(gw),
                      m.Tensor.from_numpy(np.float32([1])), keep=K, normalise=True, accumulate=False)
    got = gx.to_numpy()
    assert np.array_equal(weights.to_numpy(), want["weights"])
    assert np.array_equal(got[1:-1].reshape(x.shape), want["grad_x"]) and got[0] == 0 and got[-1] == 0


def test_ids_of_other_origin_stay_in_bounds():
    """Ids outside the experts are passed over, as those of padding rows are."""
    m = m_()
    x, _, gw = inputs(40, 20, 3, seed=13)
    chosen = np.random.RandomState(3).randint(-5, 40, (40, 3)).astype(np.int32)
    gx = m.Tensor(40, 20)
    m.router_backward(gx, m.Tensor.from_numpy(x), m.IndexTensor.from_numpy(chosen), m.IndexTensor(20), m.Tensor.from_numpy(gw), None)
    assert np.isfinite(gx.to_numpy()).all()
