"""Distillation where logits are large: masked teachers, logits with an offset, the backward alone. Bounds are those of
test_gpu_distill.py at the size of the logits' differences."""
import numpy as np
import pytest

from test_gpu_distill import check, inputs, m_, reference, run

pytestmark = pytest.mark.gpu
LOWEST = -3.4028234663852886e38
SIZES = [(5, 40, 3), (3, 1000, 8), (40, 3001, 9), (7, 20000, 20), (300, 33000, 9), (3, 70001, 30), (258, 65541, 4)]


@pytest.mark.parametrize("T", [0.5, 1.0, 4.0])
def test_teacher_rows_of_the_lowest_value(T):
    """A teacher whose entries are all the type's lowest value says that they are alike; beside larger ones that they are
    none. Their quotient by T is no number of the type where T < 1."""
    x, ids, teacher = inputs(6, 500, 7, seed=41, left_out=0)
    teacher[1] = LOWEST
    teacher[2, 3:] = LOWEST
    alike = teacher.copy()
    alike[1] = 0.0
    alike[2, 3:] = -1e6
    want, bound = reference(x, ids, alike, T=T)
    for how in ("step", "two calls"):
        check(run(m_(), x, ids, teacher, T=T, how=how), want, bound, how)
