"""What the dense products refuse (no GPU needed: an error before anything is launched)."""
import pytest
import torch


def _linear(M=4, N=8, K=16, ldx=16, ldw=16, ldr=8, ldy=8, x=4096, w=4096, y=4096, res=4096, dtype=0, act=0):
    from promoe_amd import _lib as L
    return L.lib.moe_linear(x, ldx, w, ldw, None, res, ldr, y, ldy, M, N, K, dtype, act, 0, None, 0, None)


def _gated(M=4, N=8, K=16, ldx=16, ldw=16, ldy=8, x=4096, w=4096, w2=4096, y=4096, dtype=0, act=1):
    from promoe_amd import _lib as L
    return L.lib.moe_linear_gated(x, ldx, w, w2, ldw, None, None, y, ldy, M, N, K, dtype, act, 0, None, 0, None)


BAD = [dict(M=-1), dict(N=-1), dict(K=0), dict(K=12), dict(ldx=8), dict(ldx=20), dict(ldw=8), dict(ldw=20), dict(ldy=7), dict(dtype=2),
       dict(dtype=-1), dict(act=-1), dict(act=6), dict(ldx=1 << 21), dict(ldw=1 << 21), dict(x=None), dict(w=None), dict(y=None),
       dict(x=4104), dict(w=4098)]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_c_entries_refuse(kw):
    from promoe_amd import _lib as L
    assert _linear(**kw) == L.MOE_EINVAL and b"moe_linear:" in L.lib.moe_last_error()
    assert _gated(**kw) == L.MOE_EINVAL and b"moe_linear_gated:" in L.lib.moe_last_error()


def test_c_entries_refuse_more():
    from promoe_amd import _lib as L
    assert _linear(ldr=7) == L.MOE_EINVAL
    assert _gated(w2=None) == L.MOE_EINVAL and _gated(w2=4100) == L.MOE_EINVAL
    for M, N in ((0, 8), (4, 0)):                # nothing to do
        assert _linear(M=M, N=N, ldy=8, x=None, w=None, y=None, res=None) == 0
        assert _gated(M=M, N=N, x=None, w=None, w2=None, y=None) == 0


def test_wrappers_refuse_what_is_not_on_a_gpu_or_of_another_type():
    from promoe_amd import _lib as L
    from promoe_amd import ops
    x, w = torch.zeros(2, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    with pytest.raises(L.MoeError, match="GPU"):
        ops.linear(x, w)
    with pytest.raises(L.MoeError, match="bf16 or fp16"):
        ops.linear(x.float(), w.float())
    with pytest.raises(L.MoeError, match="activations"):
        ops.linear_gated(x, w, w, act="tanh")


def test_a_result_over_an_operand_is_refused():
    """x 4 x 16 at 64 KiB, rows 32 elements apart; y elsewhere, over it, and beside its rows in the same buffer."""
    from promoe_amd import _lib as L
    X, W, R, Y = (1 << 16) * 1, (1 << 16) * 2, (1 << 16) * 3, (1 << 16) * 4

    def call(y, ldy, y32=0, res=R, ldr=32, M=4, bias=None, gated=False):
        if gated:
            return L.lib.moe_linear_gated(X, 32, W, W + (1 << 14), 32, bias, None, y, ldy, M, 8, 16, 0, 0, y32, None, 0, None)
        return L.lib.moe_linear(X, 32, W, 32, bias, res, ldr, y, ldy, M, 8, 16, 0, 0, y32, None, 0, None)

    def refused(*a, **k):
        return call(*a, **k) == L.MOE_EINVAL and b"overlaps" in L.lib.moe_last_error()

    for y, ldy, kw in ((X, 32, {}), (X + 2, 32, {}), (X + 30, 32, {}), (X + 64 - 14, 32, {}), (X + 3 * 64 + 30, 32, {}), (X - 14, 32, {}),
                       (X - 3 * 64, 32, {}), (W + 8, 32, {}), (R + 2, 32, {}), (R, 16, {}), (R, 16, dict(y32=1)), (X + 32, 40, {}),
                       (Y, 32, dict(bias=Y + 2 * 64)), (X + 32 + 2, 16, dict(y32=1)), (W + (1 << 14), 32, dict(gated=True)),
                       (Y, 32, dict(res=Y, ldr=64))):
        assert refused(y, ldy, **kw), (y - X, ldy, kw)
    if torch.cuda.is_available():
        return                                   # (what follows would launch)
    for y, ldy, kw in ((Y, 32, {}), (X + 32, 32, {}), (X + 48, 32, {}), (X + 32, 16, dict(y32=1)), (R, 32, {}), (R, 9, dict(M=1)),
                       (X + 3 * 64 + 32, 32, {}), (R + 16, 32, {}), (X - 16, 8, dict(M=1))):
        assert not refused(y, ldy, **kw), (y - X, ldy, kw)


def test_sizes_past_a_grid_are_refused():
    from promoe_amd import _lib as L
    assert _linear(M=(1 << 26) + 1) == L.MOE_EINVAL and _linear(N=(1 << 26) + 1, ldy=1 << 27, ldr=1 << 27) == L.MOE_EINVAL
    assert L.lib.moe_linear(1 << 50, 16, 1 << 51, 16, None, None, 0, 1 << 52, 1 << 26, 1 << 26, 1 << 26, 16, 0, 0, 0, None, 0, None) == L.MOE_EINVAL
    assert b"too many" in L.lib.moe_last_error()
