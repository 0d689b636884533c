"""Grouped routing over long batches (more than 2048 rows), whose choices are made in fp32 by sorted lists and handed to the 64-bit
choice where they may turn on the rounding: every form of a row, ties, masks, no numbers and near ties. A few hundred rows
against the reference and bounds of test_gpu_group_router, and all of them against calls over short batches, which choose in 64
bits alone and give the same bits."""
import numpy as np
import pytest

from test_gpu_group_router import check, inputs, m_, reference, run

pytestmark = pytest.mark.gpu


def part_of(a, rows):
    return dict(a, **{n: a[n][rows] for n in ("x", "keep", "gw") if a.get(n) is not None})


def compare(a, what="", fine=None):
    """`fine`: the rows that the reference knows; all without."""
    rows, experts = a["x"].shape
    got = run(m_(), **a)
    for half in np.array_split(np.arange(rows), 2):
        alone = run(m_(), **part_of(a, half))
        for n in alone:
            if n != "counts":
                assert np.array_equal(got[n][half], alone[n], equal_nan=n != "chosen"), f"{what} {n}"
    kept = got["chosen"][got["chosen"][:, 0] >= 0]
    assert np.array_equal(got["counts"], np.bincount(kept.reshape(-1), minlength=experts)), what
    some = np.unique(np.r_[0:20, rows - 20:rows, np.random.RandomState(60).randint(0, rows, 200)])
    some = some if fine is None else some[fine[some]]
    want, bound, whole = reference(**part_of(a, some))
    check({n: got[n][some] for n in got if n != "counts"}, want, bound, {"chosen": whole["chosen"]}, what)
    return got


# rows, experts, k, groups, open groups: all forms of a row (8 to 1024 experts), choices in one list and in up to eight, groups of one to
# three experts and of many
SIZES = [(2100, 3, 2, 3, 2), (2100, 7, 1, 7, 3), (3000, 7, 7, 1, 1), (2500, 8, 8, 4, 4), (2500, 8, 3, 4, 2), (3000, 16, 1, 1, 1),
         (2100, 16, 9, 8, 5), (2100, 15, 4, 5, 2), (2500, 30, 16, 10, 6), (2500, 32, 4, 32, 9), (2100, 60, 8, 6, 3), (2100, 60, 20, 20, 8),
         (3000, 64, 64, 1, 1), (2100, 64, 9, 64, 20), (2500, 126, 8, 42, 10), (2100, 128, 16, 64, 9), (2100, 128, 1, 8, 2),
         (2200, 250, 8, 50, 3), (2100, 256, 64, 8, 2), (2100, 300, 9, 3, 2), (2100, 512, 8, 8, 4), (2100, 510, 16, 51, 7),
         (2100, 1024, 8, 64, 8), (2100, 1024, 64, 1, 1), (2100, 1023, 9, 33, 30), (2100, 1001, 1, 1, 1)]


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, scores):
    print(f"\n[group router lists] {size} {scores}", flush=True)
    rows, experts, k, groups, opened = size
    d = inputs(rows, experts, k, seed=sum(size), std=0.1 if scores == "sigmoid" else 0.5 / experts)
    for normalise, best, keep, scale in ((True, 2, d["keep"], 2.5), (False, 1, None, 1.0)):
        a = dict(d, keep=keep, groups=groups, keep_groups=opened, best=best, scores=scores, normalise=normalise, scale=scale)
        compare(a, f"{size} {normalise}")


FORMS = [(8, 3, 4, 2), (16, 4, 4, 2), (30, 9, 5, 3), (64, 64, 1, 1), (96, 7, 8, 4), (256, 8, 8, 4), (512, 16, 1, 1), (1024, 20, 32, 3)]


@pytest.mark.parametrize("experts, k, groups, opened", FORMS)
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_ties_go_to_the_lowest_index(experts, k, groups, opened, scores):
    """Rows of ties among rows of none."""
    rows = 2300
    r = np.random.RandomState(61)
    d = inputs(rows, experts, k, seed=62)
    tied = r.uniform(size=rows) < 0.3
    d["x"][tied] = r.randint(0, 4, (tied.sum(), experts)).astype(np.float32)  # of which no two pairs have one sum
    d["x"][tied] *= np.where(r.uniform(size=(tied.sum(), experts)) < 0.1, -0.0, 1.0).astype(np.float32)
    d["x"][-1] = d["x"][3] = 0.5
    a = dict(d, bias=None, groups=groups, keep_groups=opened, scores=scores)
    compare(a, "ties")


@pytest.mark.parametrize("experts, groups", [(16, 1), (64, 1), (256, 8), (1024, 1)])
def test_choices_that_fp32_hardly_tells_apart(experts, groups):
    """Sigmoids of 1/2 and 1/2 + 2^-20 to 2^-33 around the last that is chosen, either way round and tied, with a bias as well; and so
    for the groups' sums."""
    rows, k = 4000, 3
    r = np.random.RandomState(63)
    x = np.full((rows, experts), -4.0, np.float32)
    at = np.argsort(r.uniform(size=(rows, experts)), 1)[:, :5]
    x[np.arange(rows)[:, None], at] = 4 * r.choice([-1.0, 0.0, 1.0], (rows, 5)) * 2.0 ** -r.randint(20, 34, (rows, 1))
    a = dict(x=x, k=k, gw=np.ones((rows, k), np.float32), groups=groups, keep_groups=(groups + 1) // 2)
    for bias in (None, np.full(experts, 0.25, np.float32), np.full(experts, -7.0, np.float32)):
        compare(dict(a, bias=bias), str(bias))


@pytest.mark.parametrize("experts, k, groups, opened", FORMS)
@pytest.mark.parametrize("low", [-np.inf, -3.4028234663852886e38])
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_masked_experts(experts, k, groups, opened, low, scores):
    """Experts a mask leaves out, by their logits or by a bias, come last in the order of their indices, fewer left than are chosen
    among them."""
    rows = 2200
    r = np.random.RandomState(64)
    d = inputs(rows, experts, k, seed=65)
    gone = r.uniform(size=(rows, experts)) < r.choice([0.1, 0.5, 0.9], (rows, 1))
    gone[:, -1] = False
    a = dict(d, x=np.where(gone, np.float32(low), d["x"]), bias=None, groups=groups, keep_groups=opened, scores=scores)
    compare(a, str(low))
    bias = d["bias"].copy()
    bias[::3] = -np.inf
    a = dict(d, bias=bias, groups=groups, keep_groups=opened, best=1, scores=scores, normalise=False)
    compare(a, "bias")


@pytest.mark.parametrize("experts, k, groups, opened", FORMS)
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_no_numbers(experts, k, groups, opened, scores):
    """Rows with NaN and infinities, among others that they do not touch."""
    rows = 2200
    r = np.random.RandomState(66)
    d = inputs(rows, experts, k, seed=67)
    bad = r.uniform(size=rows) < 0.1
    bad[-1] = True
    kind = r.randint(0, 4, rows)
    for i in np.flatnonzero(bad):
        some = slice(None) if kind[i] % 2 else r.randint(0, experts, 2)
        d["x"][i, some] = (np.nan, np.nan, np.inf, -np.inf)[kind[i]]
    a = dict(d, keep=None, groups=groups, keep_groups=opened, scores=scores)
    got = compare(a, scores, fine=~bad)
    assert ((got["chosen"] >= 0) & (got["chosen"] < experts)).all() and all(len(set(c)) == k for c in got["chosen"].tolist())


@pytest.mark.parametrize("experts, k, groups, opened", FORMS)
def test_logits_and_biases_of_all_sizes(experts, k, groups, opened):
    rows = 2200
    r = np.random.RandomState(68)
    d = inputs(rows, experts, k, seed=69)
    d["x"] *= r.choice([1e-30, 1e-3, 1.0, 20.0], (rows, 1)).astype(np.float32)
    d["x"][5, 0], d["x"][6, -1], d["x"][7] = 1e30, -1e30, -1e38
    for bias in (d["bias"], 1e6 * d["bias"], 1e-12 * d["bias"], 1e38 * np.sign(d["bias"])):
        for scores in ("sigmoid", "softmax"):
            a = dict(d, bias=bias.astype(np.float32), scores=scores, normalise=False, groups=groups, keep_groups=opened, gw=None)
            compare(a, f"{scores} {np.abs(bias).max()}")
