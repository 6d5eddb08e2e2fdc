"""Products in 4 bits refuse a result over the dispatch that says where it goes (no GPU needed: an error before
anything is launched)."""
from ctypes import byref

import pytest

M, N, K, E, P = 60, 30, 9984, 3, 60
X, W, S, Y, R, B, WS, XS = [i << 24 for i in range(1, 9)]
COUNTS, OFFSETS, UNITS, TOK = [(9 << 24) + (i << 16) for i in range(4)]


def experts(y, tok=TOK, y32=0):
    from promoe_amd import _lib as L
    w = L.Mx4Desc(W, S, K // 2, N * K // 2, 1 << 16)
    rc = L.lib.moe_mx4_experts(X, K, None, byref(w), None, None, None, y, N, COUNTS, OFFSETS, UNITS, E, tok, P, P, E, N, K, 0, 0, y32, None)
    return rc == L.MOE_EINVAL and b"overlaps the dispatch" in L.lib.moe_last_error()


@pytest.mark.parametrize("at,n", [(COUNTS, 4 * E), (OFFSETS, 4 * E + 4), (UNITS, 16 * E), (TOK, 4 * P)], ids=["counts", "offsets", "units", "tokens"])
def test_a_result_over_the_dispatch_is_refused(at, n):
    for y in (at, at + n - 2, at - P * N * 2 + 2):
        assert experts(y), hex(y)
    assert experts(at - P * N * 4 + 4, y32=1)
