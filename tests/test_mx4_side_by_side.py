"""Rows that lie side by side in one buffer, the same distance apart, do not overlap: products in 4 bits take them as the 16-bit ones do.

Tolerance of the values: none, the same bits as from tensors of their own."""
import pytest
import torch

X, W, S, ROW = 1 << 16, 1 << 20, 1 << 21, 4096        # a buffer with rows 4096 bytes apart, matrices elsewhere


def linear(x=X, y=X, M=4, N=8, K=64, xq=None, w=W, ldw=32, res=None, y32=0, ldy=None, ldx=ROW // 2):
    from ctypes import byref
    from promoe_amd import _lib as L
    q = L.Mx4Desc(w, S, ldw, 0, 0)
    xd = None if xq is None else L.Mx4Desc(xq, S + 65536, ROW, 0, 0)
    rc = L.lib.moe_mx4_linear(x if xq is None else None, ldx, None if xd is None else byref(xd), byref(q), None, None, None, res, ROW // 2, y,
                              ldy or ROW // (4 if y32 else 2), M, N, K, 0, 0, y32, None, 0, None)
    return rc == L.MOE_EINVAL and b"overlaps" in L.lib.moe_last_error()


def test_rows_that_touch_are_refused():
    for y in (X, X + 126, X - 14, X + 126 + ROW, X + ROW - 14, X + ROW - 2):
        assert linear(y=y), hex(y)
    assert linear(y=X + 126, y32=1) and linear(y=X - 28, y32=1)
    assert linear(y=X + 256, res=X + 270) and linear(y=X + 256, res=X + 258)      # (a residual two bytes off its result)
    assert linear(xq=X, y=X + 28) and linear(xq=X, y=X - 14)
    assert linear(y=X + 128, ldx=ROW // 2 + 8)                                   # ranges that meet, rows of another distance
    assert linear(w=W, ldw=ROW, y=W + 30, N=4) and linear(w=W, ldw=ROW, y=W - 6, N=4)


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that nothing may read: on machines without a GPU only")
def test_rows_side_by_side_are_not():
    """(no GPU: what is not refused ends at the launch)"""
    for y in (X + 128, X - 16, X + ROW - 16, X + ROW + 128):
        assert not linear(y=y), hex(y)
    assert not linear(y=X + 128, y32=1) and not linear(y=X - 32, y32=1)
    assert not linear(y=X + 256, res=X + 272) and not linear(y=X + 256, res=X + 256)
    assert not linear(xq=X, y=X + 32) and not linear(xq=X, y=X - 16)
    assert not linear(w=W, ldw=ROW, y=W + 32, N=4) and not linear(w=W, ldw=ROW, y=W - 8, N=4)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 40, 64), (5, 72, 96), (40, 136, 288), (300, 264, 544)])
def test_operands_and_results_in_one_buffer(cuda, M, N, K):
    from promoe_amd import ops
    from tests.test_mx4_gpu import matrix
    print(f"case mx4_one_buffer M={M} N={N} K={K}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(M)
    w, w2 = matrix((N, K), gen, cuda), matrix((N, K), gen, cuda)
    buf = torch.randn(M, K + 3 * N + 8, device=cuda, generator=gen).to(torch.bfloat16)
    x, res, y, tail = buf.split([K, N, N, N + 8], 1)
    y2 = tail[:, :N]
    before = buf.clone()
    want, want2 = ops.linear_mx4(x, w, residual=res), ops.linear_gated_mx4(x, w, w2)
    assert ops.linear_mx4(x, w, residual=res, out=y) is y
    ops.linear_gated_mx4(x, w, w2, out=y2)
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(y2, want2)
    assert torch.equal(x, before[:, :K]) and torch.equal(res, before[:, K: K + N]) and torch.equal(tail[:, N:], before[:, -8:])
    # rows of experts, the halves in one buffer
    E, T = 4, M
    d = ops.dispatch(torch.randint(0, E, (T, 1), device=cuda, generator=gen, dtype=torch.int32), E)
    we = matrix((E, N, K), gen, cuda)
    want = ops.experts_linear_mx4(x, we, d)
    ops.experts_linear_mx4(x, we, d, out=y)
    assert torch.equal(y, want)
