"""Moves of tokens refuse every result that lies over something that is read (no GPU needed: an error before anything is launched)."""
import pytest

T, K, H, P = 4, 2, 8, 8
X, Y, D, POS, W, N, DW = (1 << 20, 1 << 21, 1 << 22, 1 << 23, (1 << 23) + 4096, (1 << 23) + 8192, (1 << 23) + 12288)
ROW = 2 * H                                           # bytes of a row (bf16)


def sort(x=X, y=Y, pos=POS, total=N):
    from promoe_amd import _lib as L
    return L.lib.moe_sort_rows(x, H, y, H, pos, total, T, K, H, 0, None)


def unsort(x=X, y=Y, pos=POS, w=W):
    from promoe_amd import _lib as L
    return L.lib.moe_unsort_rows(x, H, y, H, pos, w, T, K, H, 0, None)


def grad(x=X, dy=D, dx=Y, pos=POS, w=W, total=N, dw=DW, h=H):
    from promoe_amd import _lib as L
    return L.lib.moe_unsort_rows_grad(dy, h, x, h, pos, w, total, dx, h, dw, T, K, h, 0, None)


def over(at, n, m):
    """Places of a result of m bytes that share the first or the last of n bytes"""
    return [at, at + n - 4, at - m + 4]


CASES = [(sort, dict(y=y)) for y in over(POS, 4 * P, P * ROW) + over(N, 4, P * ROW)]
CASES += [(unsort, dict(y=y)) for y in over(POS, 4 * P, T * ROW) + over(W, 4 * P, T * ROW)]
CASES += [(grad, dict(dx=y)) for y in over(POS, 4 * P, P * ROW) + over(W, 4 * P, P * ROW) + over(N, 4, P * ROW) + over(DW, 4 * P, P * ROW)]
CASES += [(grad, dict(dw=p)) for p in over(X, P * ROW, 4 * P) + over(D, T * ROW, 4 * P) + over(POS, 4 * P, 4 * P) + over(W, 4 * P, 4 * P) +
          over(N, 4, 4 * P) + over(Y, P * ROW, 4 * P)]
CASES += [(grad, dict(dw=p, dx=None, total=None)) for p in over(X, P * ROW, 4 * P) + over(D, T * ROW, 4 * P)]
CASES += [(grad, dict(dw=W, h=0)), (grad, dict(dw=POS + 4, h=0))]


@pytest.mark.parametrize("call,kw", CASES, ids=lambda v: v.__name__ if callable(v) else "-".join("%s=%s" % (k, v if v is None else hex(v)) for k, v in v.items()))
def test_a_result_over_what_is_read_is_refused(call, kw):
    from promoe_amd import _lib as L
    assert call(**kw) == L.MOE_EINVAL and b"overlaps" in L.lib.moe_last_error()


def test_the_gradient_of_no_tokens_is_nothing():
    from promoe_amd import _lib as L
    assert L.lib.moe_unsort_rows_grad(None, H, None, H, None, None, None, None, H, None, 0, K, H, 0, None) == 0
    assert L.lib.moe_unsort_rows_grad(D, H, X, H, POS, W, N, Y, H, DW, 0, K, H, 0, None) == 0


@pytest.mark.parametrize("dtype,h,off", [(2, 16776964, 0), (2, (1 << 24) - 4, 0), (2, 4194241, 4), (0, 4194241, 2), (1, (1 << 24) - 1, 0)])
def test_rows_of_too_many_pieces_are_refused_by_their_number(dtype, h, off):
    """One more than 65535 workgroups of 64 pieces, on 16-byte boundaries or not."""
    from promoe_amd import _lib as L
    x, y, ld = (1 << 40) + off, 1 << 42, (h + 7) // 8 * 8
    pieces = h // 4 if dtype == 2 and h % 4 == 0 and not off else h
    for rc in (L.lib.moe_sort_rows(x, ld, y, ld, POS, N, 1, 1, h, dtype, None), L.lib.moe_unsort_rows(x, ld, y, ld, POS, W, 1, 1, h, dtype, None)):
        assert rc == L.MOE_EINVAL and b"%d pieces" % pieces in L.lib.moe_last_error(), L.lib.moe_last_error()
