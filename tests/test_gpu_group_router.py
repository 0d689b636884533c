"""Routing by scores with a bias, groups and a scale (group_router_*, router_bias_update) against the formulas in 64 bits.

Tolerances, U = 2^-24. A weight is a 64-bit score rounded to fp32 (U), divided by a sum of k of them (k + 1) and times the
scale: (k + 4) U of itself. In the backward an exponential is off by (|x - top| + 5) U of itself, a sigmoid and 1 - s by 10 U,
a sum of k or of a row's 16 a lane and a tree by D = max(k, 22) more, and the products by 5: together
(4 |x - top| + 60 + 3 D) U of s (|g| + sum |g| q)."""
import numpy as np
import pytest

from util import GpuEngine, assert_bitexact

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def m_():
    return GpuEngine().m


def reference(x, k, bias=None, keep=None, groups=1, keep_groups=None, best=2, scores="sigmoid", normalise=True, scale=1.0, gw=None):
    rows, experts = x.shape
    keep_groups = groups if keep_groups is None else keep_groups
    xd = x.astype(np.float64)
    top = xd.max(1, keepdims=True)
    with np.errstate(over="ignore", invalid="ignore"):
        if scores == "sigmoid":
            e = np.exp(-np.abs(xd))
            s, rest, dist = np.where(xd < 0, e, 1.0) / (1 + e), np.where(xd < 0, 1.0, e) / (1 + e), np.zeros_like(xd)
        else:
            e = np.exp(xd - top)
            s, rest, dist = e / e.sum(1, keepdims=True), np.ones_like(xd), np.minimum(top - xd, 1e4)
    b = s + (0 if bias is None else bias.astype(np.float64))
    each = experts // groups
    if keep_groups < groups:
        score = -np.sort(-b.reshape(rows, groups, each), 2)[:, :, :best].sum(2)
        shut = np.argsort(-score, 1, kind="stable")[:, keep_groups:]
        for r in range(rows):
            for j in shut[r]:
                b[r, j * each:(j + 1) * each] = -np.inf
    order = np.argsort(-b, 1, kind="stable")[:, :k]
    if keep_groups < groups:
        # what is closed stays behind an open expert at minus infinity
        order = np.stack([[e for e in np.argsort(-b[r], kind="stable") if e // each not in shut[r]][:k] for r in range(rows)])
    kept = np.ones(rows, bool) if keep is None else keep != 0
    at = np.arange(rows)[:, None]
    picked = s[at, order]
    mass = picked.sum(1, keepdims=True)
    q = picked / mass if normalise else picked
    out = {"weights": np.where(kept[:, None], q * scale, 0)}
    bound = {"weights": (k + 4) * U * np.abs(out["weights"]) + 1e-44}
    whole = {"chosen": np.where(kept[:, None], order, -1), "counts": np.bincount(order[kept].reshape(-1), minlength=experts)}
    if gw is not None:
        g = gw.astype(np.float64)
        inner, size = (g * q).sum(1, keepdims=True), (np.abs(g) * q).sum(1, keepdims=True)
        grad, off = np.zeros_like(xd), np.zeros_like(xd)
        if scores == "softmax" and not normalise:
            grad -= s * inner
            grad[at, order] += s[at, order] * g
            off = s * size
            off[at, order] += s[at, order] * np.abs(g)
        else:
            grad[at, order] = q * rest[at, order] * (g - inner if normalise else g)
            off[at, order] = q * rest[at, order] * (np.abs(g) + size)
        far = dist if scores == "softmax" and not normalise else np.where(np.isfinite(xd), 2 * np.abs(xd), 0) * (scores == "softmax")
        out["grad_x"] = scale * grad * kept[:, None]
        bound["grad_x"] = abs(scale) * off * kept[:, None] * (4 * far.max(1, keepdims=True) + 60 + 3 * max(k, 22)) * U + 1e-44
    return out, bound, whole


def run(m, x, k, bias=None, keep=None, groups=1, keep_groups=None, best=2, scores="sigmoid", normalise=True, scale=1.0, gw=None,
        grad=None):
    rows, experts = x.shape
    tx = m.Tensor.from_numpy(x)
    tk = None if keep is None else m.IndexTensor.from_numpy(keep)
    weights, chosen, counts = m.Tensor(rows, k), m.IndexTensor(rows, k), m.IndexTensor.from_numpy(np.full(experts, 9))
    m.group_router_forward(weights, chosen, counts, tx, bias=None if bias is None else m.Tensor.from_numpy(bias), keep=tk,
                           groups=groups, keep_groups=keep_groups, group_best=best, scores=scores, normalise=normalise, scale=scale)
    got = {"weights": weights.to_numpy(), "chosen": chosen.to_numpy(), "counts": counts.to_numpy()}
    if gw is not None:
        gx = m.Tensor.from_numpy(np.full(x.shape, 7.0) if grad is None else grad)
        m.group_router_backward(gx, tx, chosen, m.Tensor.from_numpy(gw), keep=tk, scores=scores, normalise=normalise, scale=scale,
                                accumulate=grad is not None)
        got["grad_x"] = gx.to_numpy()
    return got


def check(got, want, bound, whole, what=""):
    for a, v in whole.items():
        assert np.array_equal(got[a], v), f"{what} {a}"
    for a, v in want.items():
        assert np.isfinite(got[a]).all(), f"{what} {a}: not finite"
        off = np.abs(got[a].astype(np.float64) - v)
        over = off > bound[a]
        assert not over.any(), f"{what} {a}: {over.sum()} of {over.size} beyond the bound, worst {off.max():.3g}"


def inputs(rows, experts, k, seed, std=0.1):
    r = np.random.RandomState(seed)
    x = (1.5 * r.standard_normal((rows, experts))).astype(np.float32)
    return {"x": x, "k": k, "bias": (std * r.standard_normal(experts)).astype(np.float32),
            "keep": (r.uniform(size=rows) > 0.1).astype(np.int32), "gw": r.standard_normal((rows, k)).astype(np.float32)}


# rows, experts, k, groups, open groups
SIZES = [(1, 1, 1, 1, 1), (2, 2, 1, 2, 1), (7, 3, 3, 1, 1), (64, 8, 2, 4, 2), (65, 7, 2, 7, 3), (300, 9, 4, 3, 2), (1000, 16, 4, 4, 1),
         (33, 17, 5, 1, 1), (500, 32, 8, 8, 4), (700, 60, 6, 6, 3), (129, 64, 64, 8, 8), (129, 64, 40, 8, 5), (300, 66, 8, 33, 20),
         (2000, 126, 4, 9, 5), (77, 128, 8, 64, 8), (90, 200, 16, 8, 3), (4099, 256, 8, 8, 4), (50, 258, 3, 2, 1), (40, 512, 64, 16, 4),
         (20, 1000, 10, 50, 7), (9, 1024, 64, 64, 8), (20000, 30, 2, 5, 2), (1, 1021, 7, 1, 1)]


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, scores):
    print(f"\n[group router] {size} {scores}", flush=True)
    rows, experts, k, groups, opened = size
    d = inputs(rows, experts, k, seed=sum(size), std=0.1 if scores == "sigmoid" else 0.5 / experts)
    for normalise, best, keep, scale in ((True, 2, d["keep"], 2.5), (False, 1, None, 1.0)):
        a = dict(d, keep=keep, groups=groups, keep_groups=opened, best=best, scores=scores, normalise=normalise, scale=scale)
        check(run(m_(), **a), *reference(**a), what=f"{size} {normalise}")


def test_without_a_bias():
    d = inputs(500, 40, 5, seed=1)
    for scores in ("sigmoid", "softmax"):
        a = dict(d, bias=None, scores=scores, groups=4, keep_groups=2)
        check(run(m_(), **a), *reference(**a), what=scores)


@pytest.mark.parametrize("experts, k, groups, opened", [(8, 3, 4, 2), (64, 64, 1, 1), (64, 9, 8, 3), (96, 7, 8, 4), (1024, 20, 32, 3)])
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_ties_go_to_the_lowest_index(experts, k, groups, opened, scores):
    r = np.random.RandomState(2)
    d = inputs(200, experts, k, seed=3)
    # scores of 0 to 3 have no two pairs of one sum
    d["x"] = r.randint(0, 4, (200, experts)).astype(np.float32)
    d["x"][r.uniform(size=d["x"].shape) < 0.1] = -0.0
    d["x"][3] = 0.5
    a = dict(d, bias=None, groups=groups, keep_groups=opened, scores=scores)
    check(run(m_(), **a), *reference(**a), what="ties")


def test_a_choice_that_fp32_does_not_tell_apart():
    """Two experts whose biased scores differ by 2^-30 of themselves, either way round."""
    x = np.zeros((2, 16), np.float32)
    x[:, :] = -4.0
    x[0, 3], x[1, 3] = np.float32(2 ** -28), -np.float32(2 ** -28)  # sigmoid: 1/2 +- 2^-30
    x[:, 9] = 0.0
    a = dict(x=x, k=2, bias=None, gw=np.ones((2, 2), np.float32))
    got = run(m_(), **a)
    assert got["chosen"].tolist() == [[3, 9], [9, 3]]
    b = np.full(16, 0.25, np.float32)
    assert run(m_(), **dict(a, bias=b))["chosen"].tolist() == [[3, 9], [9, 3]]


@pytest.mark.parametrize("low", [-np.inf, -3.4028234663852886e38])
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_masked_experts(low, scores):
    """Experts a mask leaves out come last, in the order of their indices, with weight and gradient 0."""
    d = inputs(100, 48, 6, seed=5)
    d["x"][:, 10:] = low
    d["x"][7, :] = low
    d["x"][7, 4] = 1.0
    a = dict(d, bias=None, scores=scores)
    check(run(m_(), **a), *reference(**a), what=str(low))


def test_a_bias_that_masks():
    d = inputs(60, 32, 4, seed=6)
    d["bias"][::2] = -np.inf
    for groups, opened in ((1, 1), (4, 2), (32, 20)):
        a = dict(d, groups=groups, keep_groups=opened, best=1)
        got, want = run(m_(), **a), reference(**a)
        check(got, *want, what=str(groups))
        assert (got["chosen"][d["keep"] != 0] % 2 == 1).all()


def test_logits_of_all_sizes():
    d = inputs(64, 24, 3, seed=7)
    d["x"] *= np.float32(40.0)
    d["x"][0, 0], d["x"][1, 1], d["x"][2] = np.float32(1e30), np.float32(-1e30), np.float32(-1e38)
    for scores in ("sigmoid", "softmax"):
        a = dict(d, scores=scores, normalise=False)
        got = run(m_(), **a)
        want, bound, whole = reference(**a)
        check({k: got[k] for k in ("weights", "chosen", "counts")}, {"weights": want["weights"]}, bound, whole, scores)
    d["x"][2, 5] = np.inf
    got = run(m_(), **dict(d, scores="sigmoid", normalise=False, bias=None, keep=None))
    assert got["chosen"][2, 0] == 5 and got["weights"][2, 0] == 1.0 and np.isfinite(got["grad_x"]).all()


@pytest.mark.parametrize("groups, opened", [(1, 1), (4, 2)])
def test_no_numbers(groups, opened):
    m = m_()
    d = inputs(6, 16, 3, seed=8)
    d["x"][1, 4] = np.nan
    d["x"][2, :] = np.nan
    d["x"][3, :] = -np.inf
    d["x"][4, 7] = np.inf
    for scores in ("sigmoid", "softmax"):
        a = dict(d, keep=None, bias=None, groups=groups, keep_groups=opened, scores=scores)
        got = run(m, **a)
        assert ((got["chosen"] >= 0) & (got["chosen"] < 16)).all()
        assert all(len(set(c)) == 3 for c in got["chosen"].tolist())
        fine = [0, 5]
        part = dict(a, x=d["x"][fine], gw=d["gw"][fine])
        want, bound, whole = reference(**part)
        check({k: got[k][fine] for k in ("weights", "chosen", "grad_x")}, want, bound, {"chosen": whole["chosen"]}, scores)
        bad = [2, 3] if scores == "sigmoid" else [1, 2, 3, 4]
        assert np.isnan(got["weights"][bad]).all()
        assert 4 not in got["chosen"][1] or scores == "softmax"
    # a chosen NaN, not normalised, is alone
    got = run(m, d["x"][1:2], 16, scores="sigmoid", normalise=False)
    assert got["chosen"][0, -1] == 4 and np.isnan(got["weights"][0, -1]) and np.isfinite(got["weights"][0, :-1]).all()


def test_padding_rows_are_left_alone():
    m = m_()
    d = inputs(40, 20, 4, seed=9)
    d["x"][d["keep"] == 0] = np.nan
    was = np.random.RandomState(10).standard_normal((40, 20)).astype(np.float32)
    for scores in ("sigmoid", "softmax"):
        for normalise in (True, False):
            a = dict(d, scores=scores, normalise=normalise)
            plain, added = run(m, **a), run(m, **a, grad=was)
            pad = d["keep"] == 0
            assert (plain["grad_x"][pad] == 0).all() and (plain["weights"][pad] == 0).all() and (plain["chosen"][pad] == -1).all()
            assert_bitexact(added["grad_x"][pad], was[pad], "padding")
            assert_bitexact(added["grad_x"][~pad], (was + plain["grad_x"])[~pad], "added")
            assert plain["counts"].sum() == 4 * (~pad).sum()
    none = run(m, **dict(d, keep=np.zeros(40, np.int32)))
    assert (none["chosen"] == -1).all() and (none["counts"] == 0).all() and (none["grad_x"] == 0).all()


@pytest.mark.parametrize("experts,k,groups,opened", [(30, 2, 5, 2), (60, 12, 1, 1), (250, 8, 5, 3)])
def test_padding_rows_of_no_choice(experts, k, groups, opened):
    """Many rows, of which padding ones hold ties, nothing or no numbers, up to the last."""
    rows = 3000
    d = inputs(rows, experts, k, seed=51)
    d["keep"][-40:] = 0
    shut = np.flatnonzero(d["keep"] == 0)
    clean = d["x"].copy()
    for i, v in enumerate((0.0, -np.inf, np.nan, np.inf)):
        d["x"][shut[i::4]] = v
    got = run(m_(), d["x"], k, d["bias"], d["keep"], groups, opened)
    want, bound, whole = reference(clean, k, d["bias"], d["keep"], groups, opened)
    check(got, want, bound, whole)


def test_choices_past_the_experts_count_as_none():
    m = m_()
    d = inputs(5, 12, 3, seed=11)
    got = run(m, d["x"], 3, scores="softmax", normalise=False)
    sel = got["chosen"].copy()
    sel[2] = [-1, 12, 0x7fffffff]
    gx = m.Tensor.from_numpy(np.full((5, 12), 7.0))
    m.group_router_backward(gx, m.Tensor.from_numpy(d["x"]), m.IndexTensor.from_numpy(sel), m.Tensor.from_numpy(d["gw"]),
                            scores="softmax", normalise=False, accumulate=False)
    assert np.isfinite(gx.to_numpy()).all() and (gx.to_numpy()[2] == 0).all()


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("normalise", [True, False])
def test_gradient_against_differences(scores, normalise):
    d = inputs(30, 20, 4, seed=12)
    a = dict(d, scores=scores, normalise=normalise, scale=1.7)
    got = run(m_(), **a)
    order, kept, at = got["chosen"], d["keep"] != 0, np.arange(30)[:, None]
    way = np.random.RandomState(13).standard_normal((30, 20))

    def value(t):  # the choice stays
        x = d["x"].astype(np.float64) + t * way
        s = 1 / (1 + np.exp(-x)) if scores == "sigmoid" else np.exp(x) / np.exp(x).sum(1, keepdims=True)
        w = s[at, order]
        w = w / w.sum(1, keepdims=True) if normalise else w
        return (1.7 * w * d["gw"])[kept].sum()

    t = 1e-4
    slope = (8 * (value(t) - value(-t)) - (value(2 * t) - value(-2 * t))) / (12 * t)
    mine = (got["grad_x"].astype(np.float64) * way).sum()
    assert abs(slope - mine) < 100 * U * np.abs(got["grad_x"] * way).sum() + 1e-9, (slope, mine)


def test_no_rows():
    m = m_()
    counts = m.IndexTensor.from_numpy(np.full(8, 5))
    m.group_router_forward(m.Tensor((0, 2)), m.IndexTensor((0, 2)), counts, m.Tensor((0, 8)))
    assert (counts.to_numpy() == 0).all()
    m.group_router_backward(m.Tensor((0, 8)), m.Tensor((0, 8)), m.IndexTensor((0, 2)), m.Tensor((0, 2)))


@pytest.mark.parametrize("experts", [1, 3, 64, 1000])
def test_bias_update(experts):
    m = m_()
    r = np.random.RandomState(experts)
    for hi in (5, 2 ** 21):
        counts, bias = r.randint(0, hi, experts).astype(np.int32), r.standard_normal(experts).astype(np.float32)
        t = m.Tensor.from_numpy(bias)
        m.router_bias_update(t, m.IndexTensor.from_numpy(counts), 0.125)
        total, c = int(counts.sum()), counts.astype(np.int64) * experts
        want = np.where(c < total, bias + np.float32(0.125), np.where(c > total, bias - np.float32(0.125), bias))
        assert_bitexact(t.to_numpy(), want, "bias")


def test_the_bias_balances():
    """Steps of the bias bring experts that are never chosen into use."""
    m = m_()
    r = np.random.RandomState(20)
    x = (0.3 * r.standard_normal((2000, 16)) + np.linspace(1, -1, 16)).astype(np.float32)
    tx, bias = m.Tensor.from_numpy(x), m.Tensor(16)
    w, chosen, counts = m.Tensor(2000, 2), m.IndexTensor(2000, 2), m.IndexTensor(16)
    first = None
    for _ in range(300):
        m.group_router_forward(w, chosen, counts, tx, bias=bias)
        first = counts.to_numpy() if first is None else first
        m.router_bias_update(bias, counts, 0.005)
    last = counts.to_numpy()
    assert first.min() == 0 and first.max() > 1000 and last.min() > 150 and last.max() < 400 and last.sum() == 4000


def test_the_same_bits_on_every_call():
    m, d = m_(), inputs(5000, 96, 6, seed=14)
    a = dict(d, groups=8, keep_groups=4)
    p, q = run(m, **a), run(m, **a)
    for k in p:
        assert np.array_equal(p[k], q[k])
