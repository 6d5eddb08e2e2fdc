"""What microscaled 4-bit floating point and its products refuse (no GPU needed: an error before anything is launched)."""
from ctypes import byref

import pytest
import torch


def desc(codes=1 << 20, scales=1 << 21, ldc=32, next_c=0, next_s=0):
    from promoe_amd import _lib as L
    return L.Mx4Desc(codes, scales, ldc, next_c, next_s)


def linear(M=4, N=8, K=64, x=1 << 16, ldx=64, xq=None, w=None, up=None, bias=None, res=None, ldr=8, y=1 << 22, ldy=8, dtype=0, act=0, y32=0):
    from promoe_amd import _lib as L
    w = desc() if w is None else w
    return L.lib.moe_mx4_linear(x, ldx, None if xq is None else byref(xq), byref(w), None if up is None else byref(up), bias, None, res, ldr, y,
                                ldy, M, N, K, dtype, act, y32, None, 0, None)


def experts(P=4, T=4, E=3, N=8, K=64, x=1 << 16, ldx=64, xq=None, w=None, up=None, y=1 << 22, ldy=8, counts=64, offsets=64, units=64,
            max_units=3, tok=None):
    from promoe_amd import _lib as L
    w = desc(next_c=256, next_s=256) if w is None else w
    return L.lib.moe_mx4_experts(x, ldx, None if xq is None else byref(xq), byref(w), None if up is None else byref(up), None, None, y, ldy,
                                 counts, offsets, units, max_units, tok, T, P, E, N, K, 0, 0, 0, None)


BAD = [dict(N=-1), dict(K=0), dict(K=48), dict(K=-32), dict(ldx=56), dict(ldx=68), dict(ldx=1 << 21), dict(ldy=7), dict(x=None), dict(x=(1 << 16) + 8),
       dict(y=None)]


@pytest.mark.parametrize("kw", BAD + [dict(M=-1), dict(dtype=2), dict(dtype=-1), dict(act=-1), dict(act=6), dict(res=1 << 23, ldr=7),
                                      dict(M=(1 << 26) + 1), dict(N=(1 << 26) + 1, ldy=1 << 27)], ids=str)
def test_linear_refuses(kw):
    from promoe_amd import _lib as L
    assert linear(**kw) == L.MOE_EINVAL and b"moe_mx4_linear:" in L.lib.moe_last_error()
    assert linear(up=desc(3 << 20, 3 << 21), **kw) == L.MOE_EINVAL


@pytest.mark.parametrize("kw", BAD + [dict(P=-1), dict(E=0), dict(E=1025), dict(T=0), dict(T=-1), dict(max_units=2), dict(counts=None),
                                      dict(offsets=None), dict(units=None)], ids=str)
def test_experts_refuse(kw):
    from promoe_amd import _lib as L
    assert experts(**kw) == L.MOE_EINVAL and b"moe_mx4_experts:" in L.lib.moe_last_error()


@pytest.mark.parametrize("kw", [dict(codes=None), dict(scales=None), dict(codes=(1 << 20) + 8), dict(scales=(1 << 21) + 2), dict(ldc=16), dict(ldc=40),
                                dict(ldc=1 << 22), dict(next_c=8), dict(next_s=2), dict(next_c=-16), dict(next_s=-4)], ids=str)
def test_descriptions_are_refused(kw):
    from promoe_amd import _lib as L
    assert linear(w=desc(**kw)) == L.MOE_EINVAL
    assert linear(up=desc(**kw)) == L.MOE_EINVAL                      # (laid out unlike the first, or not there)
    assert experts(w=desc(**kw)) == L.MOE_EINVAL
    if not any(k.startswith("next") for k in kw):                     # (rows of x have no next matrix)
        assert linear(x=None, xq=desc(**kw)) == L.MOE_EINVAL
        assert experts(x=None, xq=desc(**kw)) == L.MOE_EINVAL


def test_products_refuse_more():
    from promoe_amd import _lib as L
    assert linear(xq=desc(3 << 20, 3 << 21)) == L.MOE_EINVAL          # two x
    assert L.lib.moe_mx4_linear(1 << 16, 64, None, None, None, None, None, None, 0, 1 << 22, 8, 4, 8, 64, 0, 0, 0, None, 0, None) == L.MOE_EINVAL
    assert experts(x=1 << 50, T=1 << 24, ldx=1 << 20, tok=64) == L.MOE_EINVAL and b"2 GiB" in L.lib.moe_last_error()
    for M, N in ((0, 8), (4, 0)):                                     # nothing to do
        assert linear(M=M, N=N, x=None, y=None, w=desc(None, None)) == 0
    assert experts(P=0, T=0, x=None, y=None) == 0 and experts(N=0, ldy=0) == 0


def test_a_result_over_an_operand_is_refused():
    from promoe_amd import _lib as L
    X, W, S, Y = 1 << 16, 1 << 20, 1 << 21, 1 << 22

    def refused(rc):
        return rc == L.MOE_EINVAL and b"overlaps" in L.lib.moe_last_error()

    for y in (X, X + 3 * 128 + 126, X - 3 * 16 - 14, W, W + 7 * 32 + 30, S + 255):
        assert refused(linear(y=y)), hex(y)
    assert refused(linear(y=X - 4 * 32 + 2, y32=1))
    assert refused(linear(y=W + 6 * 32, x=None, xq=desc(W, S + 4096))) and refused(linear(y=S + 128, x=None, xq=desc(W + 4096, S)))
    assert refused(linear(bias=Y + 2)) and refused(linear(res=Y, ldr=16)) and refused(linear(res=Y, y32=1)) and refused(linear(up=desc(Y, S)))
    assert refused(experts(y=W + 2 * 256)) and refused(experts(y=S + 2 * 256 + 255))


def quantize(E=1, M=4, K=64, x=1 << 16, ldx=64, next_x=256, dtype=0, codes=1 << 20, ldc=32, next_c=128, scales=1 << 21, next_s=256, back=False):
    from promoe_amd import _lib as L
    q = desc(codes, scales, ldc, next_c, next_s)
    if back:
        return L.lib.moe_mx4_dequantize(byref(q), E, M, K, x, ldx, next_x, dtype, None)
    return L.lib.moe_mx4_quantize(x, ldx, next_x, dtype, E, M, K, byref(q), None)


@pytest.mark.parametrize("back", [False, True], ids=["quantize", "dequantize"])
@pytest.mark.parametrize("kw", [dict(M=-1), dict(E=-1), dict(K=-32), dict(K=40), dict(dtype=3), dict(dtype=-1), dict(ldx=56), dict(ldx=68), dict(ldc=16),
                                dict(ldc=40), dict(x=None), dict(codes=None), dict(scales=None), dict(x=(1 << 16) + 8), dict(codes=(1 << 20) + 4),
                                dict(E=1 << 16), dict(M=1 << 28, codes=1 << 40, scales=1 << 41), dict(codes=(1 << 16) + 16),
                                dict(scales=(1 << 16) + 512 - 4), dict(scales=(1 << 20) + 124), dict(E=2, next_x=-8), dict(E=2, next_x=4),
                                dict(E=2, next_c=-16), dict(E=2, next_c=8), dict(E=2, next_s=-1), dict(E=3, codes=(1 << 16) + 2 * 512 + 496)], ids=str)
def test_quantize_refuses(kw, back):
    from promoe_amd import _lib as L
    assert quantize(back=back, **kw) == L.MOE_EINVAL and b"quantize:" in L.lib.moe_last_error()


def test_quantize_of_nothing():
    for back in (False, True):
        assert quantize(M=0, x=None, codes=None, scales=None, back=back) == 0
        assert quantize(E=0, x=None, codes=None, scales=None, back=back) == 0


def test_bytes_of_scales():
    from promoe_amd import _lib as L
    for rows, K, n in ((0, 64, 0), (1, 32, 256), (32, 256, 256), (33, 256, 512), (33, 288, 1024), (1, 2048, 2048)):
        assert L.lib.moe_mx4_scale_bytes(rows, K) == n


def test_wrappers_refuse():
    from promoe_amd import _lib as L
    from promoe_amd import ops
    u8 = dict(dtype=torch.uint8)
    q = ops.Mx4(torch.zeros(8, 32, **u8), torch.zeros(8, 4, **u8)[:, :2])
    assert q.shape == (8, 64)
    for codes, scales in ((torch.zeros(8, 32), torch.zeros(8, 2, **u8)), (torch.zeros(8, 32, **u8), torch.zeros(8, 2)),
                          (torch.zeros(8, 24, **u8), torch.zeros(8, 1, **u8)), (torch.zeros(8, 32, **u8), torch.zeros(8, 3, **u8)),
                          (torch.zeros(8, 32, **u8), torch.zeros(7, 2, **u8)), (torch.zeros(32, **u8), torch.zeros(2, **u8)),
                          (torch.zeros(8, 0, **u8), torch.zeros(8, 0, **u8)), (torch.zeros(2, 8, 32, **u8), torch.zeros(8, 2, **u8))):
        with pytest.raises(L.MoeError, match="Mx4"):
            ops.Mx4(codes, scales)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.quantize_mx4(x), lambda: ops.linear_mx4(x, q), lambda: ops.dequantize_mx4(q)):
        with pytest.raises(L.MoeError, match="GPU"):
            call()
    with pytest.raises(L.MoeError, match="bf16, fp16 or Mx4"):
        ops.linear_mx4(x.float(), q)
    with pytest.raises(L.MoeError, match="activations"):
        ops.linear_gated_mx4(x, q, q, act="tanh")
    with pytest.raises(L.MoeError, match="Mx4"):
        ops.linear_mx4(x, torch.zeros(8, 64, dtype=torch.bfloat16))


def test_layout_of_codes_and_scales():
    """On the CPU too: rows off their boundaries are copied, scales stand in blocks of 32 rows by 8."""
    from promoe_amd import ops
    gen = torch.Generator().manual_seed(0)
    for lead, N, blocks in (((), 5, 3), ((), 32, 8), ((), 70, 17), ((3,), 33, 9), ((2,), 1, 1)):
        codes, scales = (torch.randint(0, 256, (*lead, N, n), generator=gen, dtype=torch.uint8) for n in (16 * blocks, blocks))
        for c, s in ((codes, scales), (codes.transpose(-1, -2).contiguous().transpose(-1, -2), scales),
                     (codes, scales.transpose(-1, -2).contiguous().transpose(-1, -2))):
            q = ops.Mx4(c, s)
            assert q.shape == (*lead, N, 32 * blocks) and torch.equal(q.codes, codes) and torch.equal(q.scales, scales)
            assert q.desc.ldc % 16 == 0 and q.desc.codes % 16 == 0
            flat = q.blocks.flatten(-4)
            slabs = (blocks + 7) // 8
            for r, kb in ((0, 0), (N - 1, blocks - 1), (N // 2, blocks // 2)):
                at = (r // 32 * slabs + kb // 8) * 256 + r % 32 * 8 + kb % 8
                assert torch.equal(flat[..., at], scales[..., r, kb])
    assert ops.Mx4(torch.zeros(0, 32, dtype=torch.uint8), torch.zeros(0, 2, dtype=torch.uint8)).scales.shape == (0, 2)
