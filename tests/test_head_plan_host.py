"""The vocabulary head's plan, which needs no GPU: launches within one dispatch and scratch within what the header states,
or a refusal."""
import ctypes
import random

import pytest

from mantle_amd import _lib

ITEMS = (1 << 32) - 1
G = 1 << 30


def plan(rows, dim, classes, gx, gw):
    info = _lib.mh_head_info()
    return _lib.lib().mh_plan_head(rows, dim, classes, gx, gw, ctypes.byref(info)), info


def up(v, to):
    return -(-v // to) * to


def stated(rows, dim, classes, gx, gw, info):
    """The header's bound but for the split sums, which the callers leave room for."""
    r, v, d = up(rows, 256), up(classes, 256), up(dim, 32)
    n = up(min(info.rows_at_once, rows), 256)
    total = (4 * d + 64) * (r + v) + 8 * v * n // 32 + 8 * v * n // 64 + 64 * r + (1 << 16)
    if rows <= 128:
        total += 8 * v * n // 64 + 768 * d
    if gx or gw:
        total += (4 * up(dim, 256) + 64) * (r + v) + 64 * up(dim, 256) + 8 * v * n + 64 * (n + v) + 3 * 64 * 4096 * 128
    return total


SIZES = [(1, 1, 1), (64, 128, 1000), (32768, 512, 1000), (4096, 1024, 32000), (1023, 513, 30011), (4096, 2048, 131072), (16, 4096, 32000),
         (128, 4096, 32000), (600, 4, 1 << 20), (32768, 8, 131072), (100000, 16, 70), (32768, 64, 1 << 24), (40000, 4, 1 << 26), (300, 1, (1 << 28) - (1 << 17))]


@pytest.mark.parametrize("gx, gw", [(0, 0), (1, 0), (0, 1), (1, 1)])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_launches_and_scratch(size, gx, gw):
    rc, info = plan(*size, gx, gw)
    assert rc == _lib.OK, _lib.last_error()
    assert 0 < info.largest_launch <= ITEMS
    assert 1 <= info.rows_at_once <= min(size[0], 32768)
    # split sums: a gradient's partial sums are a few of a product with fewer tiles than the chip holds, or as many
    # as its contracted axis needs
    sums = 0
    if gx:
        sums += (64 + size[2] // 65536) * up(size[1], 256) * up(info.rows_at_once, 256) * 4
    if gw:
        sums += 64 * up(size[1], 256) * up(size[2], 256) * 4
    assert info.scratch_bytes <= stated(*size, gx, gw, info) + sums


def test_rows_at_once():
    """4 GiB of logits and G, or of a forward's statistics; 256 rows at least, 32768 at most."""
    assert plan(32768, 64, 131072, 0, 0)[1].rows_at_once == 32768
    assert plan(32768, 64, 131072, 1, 1)[1].rows_at_once == 4096
    for classes in (1 << 22, 1 << 24, 1 << 26, (1 << 28) - (1 << 17)):
        for g in (0, 1):
            info = plan(32768, 4, classes, g, g)[1]
            per_row = 8 * classes if g else classes // 8
            assert info.rows_at_once * per_row <= 4 * G or info.rows_at_once == 256, (classes, g)
            assert info.rows_at_once >= 256


def test_a_forward_of_many_rows_and_classes_is_cut():
    """32768 rows against 2^24 classes at once would be a launch of 2^32 work-items."""
    rc, info = plan(32768, 64, 1 << 24, 0, 0)
    assert rc == _lib.OK and info.largest_launch <= ITEMS and info.scratch_bytes < 32 * G


def test_operands_too_large_are_refused_before_any_work():
    L = _lib.lib()
    P = ctypes.c_void_p(4096)
    for classes in (1 << 28, (1 << 31) - 1):
        for gx, gw in ((0, 0), (1, 1)):
            assert plan(300, 1, classes, gx, gw)[0] == _lib.ERR_OVERFLOW
        assert L.mh_linear_cross_entropy_fwd(P, P, P, P, P, P, 300, 1, classes) == _lib.ERR_OVERFLOW
        assert L.mh_linear_cross_entropy_bwd(P, P, P, P, P, P, P, 300, 1, classes, 0) == _lib.ERR_OVERFLOW
        assert L.mh_linear_cross_entropy_step(P, P, P, P, P, P, P, P, 300, 1, classes, 0) == _lib.ERR_OVERFLOW


def test_column_panels_are_padded_to_the_tiles_that_read_them():
    """A narrow w's column panel, whose rows are dims, is 128 of them and not 256."""
    both, forward = plan(600, 4, 1 << 20, 1, 1)[1], plan(600, 4, 1 << 20, 0, 0)[1]
    n = up(both.rows_at_once, 256)
    logits = (1 << 20) * 8 * n + 64 * (n + (1 << 20))
    assert both.scratch_bytes - forward.scratch_bytes <= logits + 128 * (4 * (1 << 20) + 64 + 4 * 768 + 64) + (64 + 16) * 128 * 768 * 4 + (1 << 20)


def test_random_sizes():
    r = random.Random(7)
    for _ in range(3000):
        size = [int(2 ** r.uniform(0, 17)), int(2 ** r.uniform(0, 13)), int(2 ** r.uniform(0, 29))]
        gx, gw = r.randint(0, 1), r.randint(0, 1)
        rc, info = plan(*size, gx, gw)
        assert rc in (_lib.OK, _lib.ERR_OVERFLOW), size
        if rc == _lib.OK:
            assert info.largest_launch <= ITEMS and info.scratch_bytes > 0, size


def test_refusals():
    for size, code in (((-1, 4, 4), _lib.ERR_INVALID), ((4, 0, 4), _lib.ERR_INVALID), ((4, 4, 1 << 31), _lib.ERR_OVERFLOW)):
        assert plan(*size, 1, 1)[0] == code
    assert _lib.lib().mh_plan_head(4, 4, 4, 0, 0, None) == _lib.ERR_NULL
    assert plan(0, 4, 4, 1, 1)[1].scratch_bytes == 0
