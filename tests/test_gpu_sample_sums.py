"""Tokens from logits whose masses strain the sums behind them (sample_tokens): far above what a workgroup looks at first, at
temperatures near the least that bins take. Against the definition in 64 bits, with the bounds of test_gpu_sample."""
import numpy as np
import pytest

from test_gpu_sample import m_, reference, run

pytestmark = pytest.mark.gpu


def check(m, x, u, T=1.0, k=0, p=1.0, mp=0.0, rows=None, what=""):
    """All rows in one call, of which those of `rows` are compared. A u of 0 lies at a border too, where the reference takes one side
    alone: a first class of less than 2^-24 may be passed over. (Below 2^-126 of the largest a mass is 0 in 32 bits, and where whole
    numbers stand for them below 2^-48 with 2^15 classes.) 2^-40 is off that border by less than any bound."""
    tok, lp = run(m, x, u, T, k, p, mp)
    for r in range(len(x)) if rows is None else rows:
        may, _ = reference(x[r], max(u[r], np.float32(2.0 ** -40)), T, k, p, mp)
        assert tok[r] in may, f"{what} row {r}: {tok[r]} and not {may}"
        assert any(abs(lp[r] - v) <= off for v, off in may[tok[r]]), f"{what} row {r}: {lp[r]} and not {may[tok[r]]}"


# rows and classes that take 64, 256, 512 and 1024 threads, none of which hold a row whole
@pytest.mark.parametrize("rows, classes", [(3000, 3001), (720, 6000), (512, 32000), (1, 32000)])
@pytest.mark.parametrize("T", [0.01, 0.0105, 0.0111, 0.02])
def test_largest_logits_far_above_the_first_at_cold_temperatures(rows, classes, T):
    """Two logits 7.9 or less above those that are looked at first, and so in their bins: up to 790 temperatures, whose
    exponential no double holds."""
    m = m_()
    r = np.random.RandomState(41)
    x = np.full((12, classes), -10.0, np.float32)
    x[:, 0] = 0.0
    x[:, classes - 7] = 7.9 - 0.25 * np.arange(12)
    x[:, classes - 9] = x[:, classes - 7] - r.choice([0.002, 0.004, 0.011], 12).astype(np.float32)
    u = r.uniform(size=12).astype(np.float32)
    u[:3] = 0.3, 0.6, 0.99
    x, u = np.tile(x, (-(-rows // 12), 1))[:rows], np.tile(u, -(-rows // 12))[:rows]
    for a in ({"p": 0.9}, {"p": 0.6}, {"k": 40, "p": 0.9}, {"k": 2, "p": 0.55}, {"k": 1}, {"k": 2}, {"p": 0.9, "mp": 0.5}):
        for v in {0.3, 0.7} if rows == 1 else {None}:
            check(m, x, u if v is None else np.float32([v]), T=T, **a, rows=range(min(rows, 24)), what=str(a))


LOG2E = float(np.float32(1.4426950408889634))  # a temperature at which x of -n has a mass of 2^-n, but for 2^-26 n of it


@pytest.mark.parametrize("classes, step", [(7000, 256), (32000, 256), (131072, 512)])
def test_a_goal_where_sums_round_apart(classes, step):
    """Masses of 1, 2^-53, 2^-53, a half and a half, `step` classes or a wavefront apart: the sum of the first three is 1 from the
    left and 1 + 2^-52 from the right, and u = 1/2 of their total lies between. Far from it, behind it, is the last class."""
    m = m_()
    x = np.full((1, classes), -np.inf, np.float32)
    x[0, 0], x[0, step], x[0, 2 * step] = 0, -53, -53
    x[0, 3 * step] = x[0, 3 * step + 200] = -1
    for a in ({}, {"mp": 2.0 ** -60}, {"k": 6}):
        check(m, x, np.float32([0.5]), T=LOG2E, **a, what=str(a))


@pytest.mark.parametrize("rows, classes", [(1, 900), (1, 7000), (1, 32000), (1, 131072), (300, 900), (720, 6000), (512, 32000), (2, 600001)])
def test_masses_of_powers_of_two(rows, classes):
    """A few classes of 1 to 2^-60 in a row of none, where a u of eighths meets the borders of their sums."""
    m = m_()
    r = np.random.RandomState(42)
    for turn in range(20 if rows == 1 else 2):
        x = np.full((rows, classes), -np.inf, np.float32)
        for row in x:
            some = np.unique(r.choice([1, 4, 64, 256, 512, 1024]) * r.randint(0, classes // 1024 + 1 if r.randint(2) else 1 + classes // 4, 12) % classes)
            row[some] = -r.choice([0, 0, 1, 2, 52, 53, 54, 60], len(some))
        x[0, 0] = 0
        u = (r.randint(0, 9, rows) / 8).astype(np.float32)
        for a in ({}, {"k": 900}, {"p": 0.75}):
            check(m, x, u, T=LOG2E, **a, rows=range(min(rows, 30)), what=str(a))


@pytest.mark.parametrize("classes", [900, 32000, 131072, 600001])
def test_the_last_class_that_is_kept(classes):
    """u just below 1 where nothing behind the first classes is kept."""
    m = m_()
    r = np.random.RandomState(43)
    x = (0.1 * r.standard_normal((4, classes))).astype(np.float32)
    x[:, :3] = [7.0, 7.1, 6.9]
    for a in ({"k": 3}, {"mp": 0.5}, {"k": 3, "p": 0.9999}):
        tok, _ = run(m, x, np.full(4, 1 - 2.0 ** -24, np.float32), **a)
        assert (tok == 2).all(), (a, tok)


# How many logits lie how many 64ths below the largest. In 512 and 1024 threads' sums half of the mass ends, by rounding, behind a
# thread's last class, where its bins are empty; in the first row it begins again two threads on.
HALVES = [(7000, {0: 1, 10: 8, 22: 1, 1: 1, 8: 2, 4: 8, 9: 5, 12: 5, 3: 4, 23: 2, 29: 5, 41: 307, 47: 1, 75: 1, 127: 1, 151: 1, 216: 1,
                  240: 1, 302: 1, 349: 1, 401: 1, 435: 1, 483: 1, 548: 1}),
          (32000, {0: 2, 13: 1, 8: 10, 15: 11, 9: 4, 11: 9, 6: 10, 4: 7, 3: 1, 10: 9, 17: 5, 16: 1, 1: 5, 12: 1, 7: 5, 2: 2, 18: 1,
                   41: 654, 43: 1, 113: 1, 163: 1, 188: 1, 258: 1, 289: 1, 342: 1, 432: 1, 469: 1, 517: 1, 544: 1})]


@pytest.mark.parametrize("classes, bins", HALVES, ids=lambda v: str(v) if isinstance(v, int) else "")
def test_a_cut_where_sums_round_apart(classes, bins):
    m = m_()
    x = np.full((1, classes), -np.inf, np.float32)
    some = np.repeat([-k / 64 for k in bins], list(bins.values()))
    for order in (some, some[::-1]):
        x[0, :len(some)] = order
        for a in ({}, {"k": len(some) + 7}, {"mp": 1e-3}):
            for u in (0.0, 0.3, 0.77, 1 - 2.0 ** -24):
                check(m, x, np.float32([u]), T=0.25, p=0.5, **a, what=f"{a} {u}")


def test_a_bulk_of_classes_far_below_the_largest():
    """2^24 classes of which all but the first have e^-26.9 = 2^-38.8 of its mass, 2^-14.8 together; u draws among them, and top_p's
    border lies there. A class' mass is off by (26.9 + 4) 2^-24 of itself, and so the bulk's, a place by as much of what lies
    behind it; u and top_p are exact."""
    m = m_()
    n = 1 << 24
    x = np.full((1, n), -26.9, np.float32)
    x[0, 0] = 0.0
    each = np.exp(np.float64(x[0, 1]))
    off = (26.9 + 4) * 2.0 ** -24
    for behind in (2.0 ** -15.5, 2.0 ** -16, 2.0 ** -18):
        u = np.float32(1 - behind)
        for k in (n - 1, n - 12345):
            total = 1 + (k - 1) * each
            tok, lp = run(m, x, np.float32([u]), k=k)
            left = (1 - np.float64(u)) * total / each  # classes behind the one that is drawn
            assert abs(k - left - tok[0]) <= off * left + 2, (behind, k, tok)
            assert abs(lp[0] + 26.9 + np.log(total)) <= 1e-5
    p = np.float32(1 - 2.0 ** -16)
    tok, lp = run(m, x, np.float32([1 - 2.0 ** -24]), p=p)
    total = 1 + (n - 1) * each
    kept = n - (1 - np.float64(p)) * total / each
    left = 2.0 ** -24 * total / each
    assert abs(kept - left - tok[0]) <= off * (n - kept + left) + 3, tok


@pytest.mark.parametrize("rows, classes", [(300, 900), (720, 6000), (512, 32000), (1, 32000), (3, 600001)])
@pytest.mark.parametrize("T", [0.01, 0.3, LOG2E])
def test_the_same_tokens_on_every_call(rows, classes, T):
    """Where sums round apart too: logits of 1 to 60 temperatures, the rows again and again."""
    m = m_()
    r = np.random.RandomState(44)
    x = np.full((rows, classes), -np.inf, np.float32)
    for row in x:
        some = r.randint(0, classes, 700)
        row[some] = -np.float32(T) * r.choice([0, 1, 2, 30, 36, 37, 38, 60], len(some))
    x[:, 0] = 0
    u = r.randint(0, 9, rows).astype(np.float32) / 8
    for a in ({"p": 0.75}, {"k": 500, "p": 0.75}, {"k": 500}):
        seen = [run(m, x, u, T=T, **a) for _ in range(4)]
        assert all(np.array_equal(tok, seen[0][0]) and np.array_equal(lp, seen[0][1]) for tok, lp in seen)
