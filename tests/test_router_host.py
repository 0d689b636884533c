"""Refusals of the router that need no GPU. The addresses are never read."""
import ctypes

from mantle_amd import _lib


def test_rows_whose_choices_pass_64_bits():
    L, P = _lib.lib(), ctypes.c_void_p(4096)
    for rows, k in ((1 << 62, 4), (1 << 60, 16), ((1 << 63) - 1, 64), ((1 << 31) // 8, 8)):
        assert L.mh_router_fwd(P, P, P, P, P, None, rows, 64, k, 0) == _lib.ERR_OVERFLOW
        assert L.mh_router_bwd(P, P, None, P, P, P, P, rows, 64, k, 0, 0) == _lib.ERR_OVERFLOW
