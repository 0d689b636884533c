"""Tokens from logits (sample_tokens) against the definition in 64 bits.

A mass is off by D = (|x - max| / T + 4) 2^-24 of itself (the difference's rounding, an exponential) and 2^-shift of the largest, so
a row's shares by delta = the mean of D over what is kept, twice. Where a cut or u lies within that of a border either side of
it is right, so a row has a set of right tokens; rows whose set has more than one are counted, and may be one in fifty."""
import numpy as np
import pytest

from util import GpuEngine

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def m_():
    return GpuEngine().m


def reference(x, u, T=1.0, k=0, p=1.0, mp=0.0):
    """One row: {token: [(logprob, its bound)]} for every cut and every u within the rounding, nearly always a single one, and
    what is kept."""
    x = (x + np.float32(0)).astype(np.float64)
    n = len(x)
    if np.isnan(x).any() or x.max() == -np.inf:
        return {-1: [(np.nan, 0.0)]}, np.zeros(n, bool)
    top = x.max()
    if not T > 0:
        return {int(np.argmax(x)): [(0.0, 0.0)]}, np.arange(n) == np.argmax(x)
    T = float(np.float32(T))
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        y = np.where(x == top, 0.0, (x - top) / T if np.isfinite(T) else np.where(x == -np.inf, -np.inf, 0.0))
        e = np.exp(y)
        rel = np.where(e > 0, np.minimum(np.abs(y), 1e3) + 4, 0) * U
    order = np.argsort(-x, kind="stable")
    least = most = k if 0 < k < n else n
    if p < 1:
        p = max(float(np.float32(p)), 0.0)
        m = np.where(np.arange(n) < most, e[order], 0.0)
        total = m.sum()
        share = np.cumsum(m) / total
        # equal masses have exact sums
        delta = 1e-15 if same(m) else 2 * (m * rel[order]).sum() / total + n * 2.0 ** -45
        least, most = (max(1, min(most, int((share < p + d).sum()) + 1)) for d in (-delta, delta))
        if p == 0:
            least = most = 1
        if same(m):  # a share of p itself ends the cut
            most = least
    if mp > 0:
        mp = float(np.float32(mp))
        edge = T * np.log(min(mp, 1.0))
        many = [max(1, int(((x == top) | (x - (top if top < np.inf else 0.0) >= edge + d * abs(edge))).sum())) for d in (1e-14, -1e-14)]
        many = [int((x == top).sum())] * 2 if top == np.inf else many
        least, most = min(least, many[0]), min(most, many[1])
    u = min(max(float(u), 0.0), 1 - U) if u == u else 0.0
    may = {}
    for count in range(least, most + 1):
        keep = np.zeros(n, bool)
        keep[order[:count]] = True
        q = np.where(keep, e, 0.0)
        total = q.sum()
        share = np.cumsum(q) / total
        off = 2 * (q * rel).sum() / total + n * 2.0 ** -45
        delta = 0.0 if same(q) and u * len(q[q > 0]) % 1 == 0 else off
        last = int(np.flatnonzero(q)[-1])
        lo, hi = (min(int((share <= u + d).sum()), last) for d in ((-delta, delta) if u > 0 else (0.0, 0.0)))
        for at in lo + np.flatnonzero(q[lo:hi + 1] > 0):
            at = int(at)
            lp = np.log(q[at] / total)
            may.setdefault(at, []).append((lp, off + rel[at] + 2 * U * abs(lp) + 1e-44))
    return may, keep


def same(q):
    return len(set(q[q > 0])) == 1


def run(m, x, u, T=None, k=None, p=None, mp=None, logprob=True):
    rows = len(x)
    f = lambda a: None if a is None else m.Tensor.from_numpy(np.broadcast_to(np.float32(a), (rows,)))  # noqa: E731
    tok, lp = m.IndexTensor.from_numpy(np.full(rows, 77)), m.Tensor.from_numpy(np.full(rows, 77.0))
    m.sample_tokens(tok, m.Tensor.from_numpy(x), m.Tensor.from_numpy(np.float32(u)), temperature=f(T),
                    top_k=None if k is None else m.IndexTensor.from_numpy(np.broadcast_to(np.int32(k), (rows,))), top_p=f(p),
                    min_p=f(mp), logprob=lp if logprob else None)
    return tok.to_numpy(), lp.to_numpy()


def check(m, x, u, T=None, k=None, p=None, mp=None, unsure=None, what=""):
    got, lp = run(m, x, u, T, k, p, mp)
    rows = len(x)
    left = 0
    at = lambda a, d, r: d if a is None else np.broadcast_to(a, (rows,))[r]  # noqa: E731
    for r in range(rows):
        may, _ = reference(x[r], np.float32(u[r]), at(T, 1.0, r), int(at(k, 0, r)), at(p, 1.0, r), at(mp, 0.0, r))
        left += len(may) > 1
        assert got[r] in may, f"{what} row {r}: {got[r]} and not {may}"
        right = [np.isnan(lp[r]) if np.isnan(v) else abs(lp[r] - v) <= off for v, off in may[got[r]]]
        assert any(right), f"{what} row {r}: {lp[r]} and not {may[got[r]]}"
    assert left <= (rows / 50 if unsure is None else unsure), f"{what}: {left} of {rows} rows are too near a border"


def logits(rows, classes, seed, std=2.0):
    r = np.random.RandomState(seed)
    x = std * r.standard_normal((rows, classes))
    for i in range(rows):
        x[i, r.randint(0, classes, 8)] += r.uniform(2, 10, 8)
    return x.astype(np.float32), r.uniform(size=rows).astype(np.float32)


SIZES = [(1, 1), (3, 2), (50, 3), (40, 7), (30, 64), (30, 65), (20, 1000), (9, 1023), (9, 1025), (7, 4096), (33, 5001), (5, 30011),
         (3, 32000), (4, 65536), (3, 70001), (2, 131072), (2, 200003)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size):
    print(f"\n[sample] {size}", flush=True)
    m = m_()
    x, u = logits(*size, seed=sum(size))
    r = np.random.RandomState(1)
    rows = size[0]
    check(m, x, u, unsure=1, what="as they are")
    for k in (1, 2, 50, size[1] // 2, size[1], size[1] + 5):
        check(m, x, u, T=0.7, k=k, unsure=1, what=f"top_k {k}")
    for p in (0.0, 0.3, 0.9, 0.999):
        check(m, x, u, T=1.3, p=p, unsure=1, what=f"top_p {p}")
    for mp in (0.01, 0.5, 1.0, 2.0):
        check(m, x, u, mp=mp, unsure=0, what=f"min_p {mp}")
    check(m, x, u, T=r.choice([0.0, 0.5, 1.0, 2.0, 50.0], rows), k=r.choice([-1, 0, 3, 40], rows), p=r.choice([1.0, 0.8, 0.5], rows),
          mp=r.choice([0.0, 0.05, -1.0], rows), unsure=1, what="mixed")


@pytest.mark.parametrize("size", [(257, 9000), (300, 40001)], ids=str)
def test_many_rows_of_many_classes(size):
    m = m_()
    x, u = logits(*size, seed=sum(size))
    r = np.random.RandomState(1)
    rows = size[0]
    check(m, x, u, T=r.choice([0.0, 0.5, 1.0, 1.4], rows), k=r.choice([0, 1, 40, 700], rows), p=r.choice([1.0, 0.95, 0.6], rows),
          mp=r.choice([0.0, 0.03], rows), what="mixed")


@pytest.mark.parametrize("classes", [(1 << 19) + 1, 700001])
def test_more_classes_than_bins_count(classes):
    m = m_()
    x, u = logits(2, classes, seed=21)
    for a in ({}, {"k": 50}, {"p": 0.9, "T": 0.7}, {"T": 0.0}, {"k": 1000, "p": 0.8, "mp": 0.01}):
        check(m, x, u, **a, unsure=1, what=str(a))


@pytest.mark.parametrize("rows, classes", [(3, 100000), (260, 40000)])
def test_a_logit_far_above_those_before_it(rows, classes):
    """One that lies beyond what a workgroup holds, by a little or by more than any bin."""
    m = m_()
    x, u = logits(rows, classes, seed=22)
    for above in (5.0, 12.0, 40.0, 1e4):
        x[:, classes - 7] = x.max() + above
        x[:, classes - 300] = x.max() - 0.5
        check(m, x, u, k=40, p=0.99, what=f"+{above}")
        # shares of 1 / 20000 or so against borders of 2 delta, 1e-6: one row in thirty or so
        check(m, x, u, T=3.0, p=0.5, unsure=rows / 20 + 1, what=f"+{above}, warm")


@pytest.mark.parametrize("rows", [3, 300])
def test_largest_logits_last(rows):
    """Classes by rising logits, close together: the largest lie behind all that is looked at first, and bins begin among them."""
    m = m_()
    r = np.random.RandomState(31)
    x = np.sort(1e-5 * r.standard_normal((rows, 120001)).astype(np.float32), axis=1)
    x[3:] = -np.inf
    x[3:, 7] = 1.0
    u = r.uniform(size=rows).astype(np.float32)
    for a in ({"k": 50000, "p": 0.4}, {"p": 0.02}, {"k": 900, "p": 0.6}, {"k": 70001}, {"p": 0.7, "T": 0.02}):
        check(m, x, u, **a, unsure=3, what=str(a))


def test_many_logits_at_the_edge_of_a_bin():
    """Thousands within 2^-24 of a bin's edge, and more above the first look's largest: which bin is theirs may not turn on
    how far from the edge the bins begin."""
    m = m_()
    r = np.random.RandomState(32)
    n = 120001
    # top_p ends among some 50000, top_k among as many behind them
    x = (-2.0 ** -15 - 7e-6 * r.uniform(size=(2, n)) - np.where(r.uniform(size=(2, n)) < 0.5, 1.6e-5, 0.0)).astype(np.float32)
    for row in x:
        some = r.permutation(n)[:6000]
        row[some] = (-2.0 ** -15 * (1 - np.arange(1, 6001) * 2.0 ** -24)).astype(np.float32)
        row[0] = 0.0
        for at in range(5000, n, 7680):
            row[at:at + 100] = (1e-6 * r.uniform(1, 2, 100)).astype(np.float32)
    for u in (0.2, 0.55, 0.91):
        check(m, x, np.float32([u, u + 0.03]), k=90000, p=0.3, unsure=2, what=str(u))


@pytest.mark.parametrize("std", [1e-5, 0.01, 0.2])
def test_logits_close_together(std):
    """Thousands of classes in a bin: narrower ones, or where they are too close for any, the search over their bits."""
    m = m_()
    r = np.random.RandomState(23)
    x = (std * r.standard_normal((4, 70000))).astype(np.float32)
    u = r.uniform(size=4).astype(np.float32)
    for a in ({"k": 30000}, {"p": 0.5}, {"k": 50000, "p": 0.4}, {"T": 0.05, "p": 0.9}, {"T": 20.0, "k": 100, "p": 0.3}):
        check(m, x, u, **a, unsure=4, what=f"{std} {a}")


@pytest.mark.parametrize("T", [0.005, 0.01, 0.02, 0.1])
def test_cold(T):
    """Cuts far below the largest, where masses are nothing."""
    m = m_()
    x, u = logits(6, 5000, seed=24)
    for a in ({"k": 1}, {"k": 60}, {"k": 3000}, {"p": 0.9999}, {"k": 500, "p": 0.999999}):
        check(m, x, u, T=T, **a, unsure=2, what=f"{T} {a}")


@pytest.mark.parametrize("rows", [12, 720, 3000])
@pytest.mark.parametrize("kind", ["few", "ties", "close", "masked", "far"])
def test_many_rows_take_other_workgroups(rows, kind):
    """The same 12 rows over and over, which fewer threads a row take where there are many of them."""
    m = m_()
    x, u = logits(12, 3001, seed=25)
    r = np.random.RandomState(26)
    if kind == "ties":
        x = np.round(x)
    if kind == "close":
        x = (1e-3 * r.standard_normal(x.shape)).astype(np.float32)
    if kind == "masked":
        x[:, 5:2900] = -np.inf
        x[1], x[2, 7], x[3, 2950] = -np.inf, np.nan, np.inf
    if kind == "far":
        x[:, -2] = x.max() + np.float32([3, 9, 30] * 4)
    for a in ({}, {"k": 7}, {"k": 1500}, {"p": 0.7}, {"k": 900, "p": 0.9, "mp": 1e-3, "T": 1.2}, {"T": 0.0}, {"T": 0.1, "p": 0.99}, {"T": 8.0, "k": 2000, "p": 0.8}):
        check(m, x, u, **a, unsure=12, what=f"{kind} {a}")
        tok, lp = run(m, x, u, **a)
        many = run(m, np.tile(x, (rows // 12, 1)), np.tile(u, rows // 12), **a)
        right = [reference(x[i], u[i], a.get("T", 1.0), a.get("k", 0), a.get("p", 1.0), a.get("mp", 0.0))[0] for i in range(12)]
        for i in range(12):
            assert len(set(many[0][i::12].tolist())) == 1
            t, l = int(many[0][i]), many[1][i]
            assert t in right[i] and any(np.isnan(l) and np.isnan(v) or abs(l - v) <= off for v, off in right[i][t]), f"{kind} {a} {i}"


def test_many_rows():
    m = m_()
    x, u = logits(6000, 40, seed=2)
    r = np.random.RandomState(3)
    check(m, x, u, T=r.choice([0.0, 0.5, 1.0, 2.0], 6000), k=r.choice([0, 1, 5, 30], 6000), p=r.choice([1.0, 0.9, 0.3], 6000),
          mp=r.choice([0.0, 0.1], 6000), unsure=20, what="rows")


@pytest.mark.parametrize("classes", [40, 3000, 40000])
def test_ties(classes):
    """Logits of a few values: the lowest indices stay where a cut falls among equals, and sums of equals are exact."""
    m = m_()
    r = np.random.RandomState(4)
    rows = 24
    x = r.randint(0, 3, (rows, classes)).astype(np.float32)
    x[0] = 1.0
    x[1] = -0.0
    x[1, ::2] = 0.0
    u = r.uniform(size=rows).astype(np.float32)
    for k in (1, 2, 7, classes // 2, classes - 1):
        check(m, x, u, k=k, unsure=1, what=f"top_k {k}")
    check(m, x, u, T=0.5, p=0.61803, unsure=2, what="top_p")
    check(m, x, u, T=0.5, k=classes // 3, p=0.61803, unsure=2, what="both")
    # halves and quarters of equal classes
    y = np.zeros((4, classes), np.float32)
    for p, many in ((0.5, classes // 2), (0.25, classes // 4), (0.75, classes * 3 // 4)):
        tok, lp = run(m, y, [0.0, 0.5, 0.99, 1 - U], p=p)
        assert tok.max() < many and tok[0] == 0 and tok[1] == many // 2 and tok[3] == many - 1
        assert np.allclose(lp, -np.log(many), rtol=1e-6)


def test_borders_of_u():
    """u of 0 draws the first class that is kept, u just below 1 the last; out of range it is held to them."""
    m = m_()
    x, _ = logits(6, 500, seed=5)
    x[:, 0] = x[:, -1] = -np.inf
    for u, last in ((0.0, False), (-3.0, False), (np.nan, False), (1 - U, True), (1.0, True), (9.0, True), (np.inf, True)):
        for k in (0, 5):
            tok, _ = run(m, x, np.full(6, u, np.float32), k=k)
            for r in range(6):
                keep = reference(x[r], 0.5, 1.0, k)[1] & (x[r] > -np.inf)
                at = np.flatnonzero(keep)
                if last and k == 0:  # what is beyond the last 2^-24 of the mass
                    assert keep[tok[r]] and np.exp(x[r, tok[r] + 1:].astype(np.float64)).sum() <= 4 * U * np.exp(x[r].astype(np.float64)).sum()
                else:
                    assert tok[r] == (at[-1] if last else at[0])


def test_uniform_over_a_grid_of_u():
    """Every u of a grid draws its own share."""
    m = m_()
    x, _ = logits(1, 30, seed=6)
    n = 5000
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    check(m, np.repeat(x, n, 0), u, T=1.5, unsure=3, what="grid")
    check(m, np.repeat(x, n, 0), u, T=1.5, k=6, p=0.95, unsure=3, what="grid cut")


@pytest.mark.parametrize("classes", [6, 100, 5000, 70000])
def test_masks_and_no_numbers(classes):
    m = m_()
    x, u = logits(8, classes, seed=7)
    x[0, 1:] = -np.inf
    x[1, :] = -np.inf
    x[2, classes // 2] = np.nan
    x[3, :] = np.nan
    x[4, 3] = np.inf
    x[5, 2] = x[5, 5] = np.inf
    x[6, :-1] = -3.4028234663852886e38
    x[7, ::2] = -np.inf
    for a in ({}, {"k": 3}, {"p": 0.7}, {"mp": 0.2}, {"T": 0.0}, {"T": 0.3, "k": 3, "p": 0.9, "mp": 0.1}, {"k": classes}):
        check(m, x, u, **a, unsure=0, what=str(a))


@pytest.mark.parametrize("T", [1e-45, 1e-30, 1e-3, 1e3, 1e30, np.inf, -1.0, np.nan, -np.inf, 0.0])
def test_temperatures(T):
    m = m_()
    x, u = logits(12, 300, seed=8)
    x[0, :3] = x[0].max()
    x[1, 10] = -np.inf
    check(m, x, u, T=T, unsure=0, what=str(T))
    check(m, x, u, T=T, k=9, unsure=0, what=f"{T} top_k")


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, -1.0, 0.0])
def test_settings_out_of_range(value):
    m = m_()
    x, u = logits(12, 300, seed=9)
    as_p = value if value <= 0 else 1.0
    got = run(m, x, u, p=value, mp=0.0)
    want = run(m, x, u, p=as_p, mp=0.0)
    assert np.array_equal(got[0], want[0])
    if value <= 0:
        assert np.array_equal(got[0], x.argmax(1)) and (got[1] == 0).all()
    as_mp = value if value > 0 else 0.0
    assert np.array_equal(run(m, x, u, mp=value)[0], run(m, x, u, mp=as_mp)[0])
    if value > 1:
        assert np.array_equal(run(m, x, u, mp=value)[0], x.argmax(1))


def test_logits_of_all_sizes():
    m = m_()
    x, u = logits(20, 200, seed=10)
    for by in (1e-38, 1e-6, 1e6, 1e36):
        check(m, (x * np.float32(by)).astype(np.float32), u, k=50, p=0.9, unsure=8, what=str(by))
    check(m, x + np.float32(30000.0), u, p=0.9, unsure=1, what="offset")


def test_without_a_logprob_and_in_one_call():
    m = m_()
    x, u = logits(30, 900, seed=11)
    a = dict(T=0.8, k=40, p=0.9, mp=0.01)
    tok, _ = run(m, x, u, **a)
    assert np.array_equal(tok, run(m, x, u, **a, logprob=False)[0])
    for r in (0, 13, 29):  # a row does not depend on its neighbours
        one = run(m, x[r:r + 1], u[r:r + 1], **a)
        assert one[0][0] == tok[r]


def test_the_same_bits_on_every_call():
    m = m_()
    x, u = logits(40, 50000, seed=12)
    a = run(m, x, u, T=1.4, p=0.97)
    for _ in range(3):
        b = run(m, x, u, T=1.4, p=0.97)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_no_rows():
    m = m_()
    m.sample_tokens(m.IndexTensor((0,)), m.Tensor((0, 5)), m.Tensor((0,)))
