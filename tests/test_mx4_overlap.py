"""Products in 4 bits refuse a result over the dispatch that says where it goes, and a workspace over anything else (no GPU needed: an error
before anything is launched)."""
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


def linear(ws, quantised=False, gated=False, y=Y):
    from promoe_amd import _lib as L
    need = L.lib.moe_mx4_linear_workspace_bytes(M, N, K, quantised, gated)
    assert need > 0
    w, up, x = L.Mx4Desc(W, S, K // 2, 0, 0), L.Mx4Desc(W + (1 << 22), S + (1 << 22), K // 2, 0, 0), L.Mx4Desc(X, XS, K // 2, 0, 0)
    rc = L.lib.moe_mx4_linear(None if quantised else X, K, byref(x) if quantised else None, byref(w), byref(up) if gated else None, B,
                              B + 4096 if gated else None, None if gated else R, N, y, N, M, N, K, 0, 0, 0, ws, need, None)
    return rc == L.MOE_EINVAL and b"the workspace overlaps" in L.lib.moe_last_error()


@pytest.mark.parametrize("at,n,kw", [(X, M * K * 2, {}), (X, M * K // 2, dict(quantised=True)), (XS, 2 * 39 * 256, dict(quantised=True)), (W, N * K // 2, {}),
                                     (S, 39 * 256, {}), (B, 2 * N, {}), (R, M * N * 2, {}), (Y, M * N * 2, {}), (W + (1 << 22), N * K // 2, dict(gated=True)),
                                     (S + (1 << 22), 39 * 256, dict(gated=True)), (B + 4096, 2 * N, dict(gated=True))])
def test_a_workspace_over_anything_is_refused(at, n, kw):
    from promoe_amd import _lib as L
    need = L.lib.moe_mx4_linear_workspace_bytes(M, N, K, kw.get("quantised", False), kw.get("gated", False))
    for ws in (at, (at + n - 2) // 16 * 16, (at - need + 16) // 16 * 16):
        assert linear(ws, **kw), hex(ws)
