"""Tokens from logits whose masses strain the sums behind them (sample_tokens): far above what a workgroup looks at first, at
temperatures near the least that bins take. Against the definition in 64 bits, with the bounds of test_gpu_sample."""
import numpy as np
import pytest

from test_gpu_sample import m_, reference, run

pytestmark = pytest.mark.gpu


def check(m, x, u, T=1.0, k=0, p=1.0, mp=0.0, rows=None, what=""):
    """All rows in one call, of which those of `rows` are compared."""
    tok, lp = run(m, x, u, T, k, p, mp)
    for r in range(len(x)) if rows is None else rows:
        may, _ = reference(x[r], u[r], T, k, p, mp)
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
