"""Microscaled 4-bit floating point on the GPU against the definition in 64 bits.

Quantising and its way back are exact: codes and scales are compared as they are.  Tolerance of an element of a product: as for products of
16-bit values (test_linear_gpu.py), a sum goes through blocks of at least 8 in the matrix core and then at most K / 8 + 8 additions that
round (or cut) by at most 2^-23 of what is added up so far; an fp16 x goes as two bf16 parts, which are at most 1 + 2^-7 of it together, and
so through twice as many.  With e = (K / 4 + 40) 2^-23 (1 + 2^-7) sum |x w| for all, the activation passes on its slope times e and adds
(8 + |v|) 2^-23 |v|; the rounding to the result's type is half a step: 2^-8 (bf16), 2^-11 (fp16), 2^-24 (fp32) of the value."""
import pytest
import torch

from tests.test_linear_gpu import ACTS, act64, check, rows, slope

pytestmark = pytest.mark.gpu
GRID = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def values(codes, scales):
    """64-bit values of codes [..., K / 2] and scales [..., K / 32]"""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return GRID.to(codes.device)[c.long()] * s.repeat_interleave(32, -1)


def quantised(x):
    """(codes, scales) of x by the definition, in 64 bits"""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    fine = torch.isfinite(b).all(-1)
    e = torch.where(fine & (top > 0), torch.frexp(torch.where(fine, top, 1.0)).exponent - 1, -200)
    byte = torch.where(fine, (e - 2).clamp(min=-127) + 127, 255)
    r = (b.abs() / torch.exp2(byte.double() - 127)[..., None]).nan_to_num(0.0, 7.0)
    n = torch.zeros_like(r, dtype=torch.uint8)
    for border, down in ((.25, 1), (.75, 0), (1.25, 1), (1.75, 0), (2.5, 1), (3.5, 0), (5.0, 1)):
        n += (r > border) if down else (r >= border)
    n = (n + 8 * torch.signbit(x).unflatten(-1, (-1, 32)).to(torch.uint8)).flatten(-2)
    return n[..., 0::2] | n[..., 1::2] << 4, byte.to(torch.uint8)


def same(q, x):
    codes, scales = quantised(x)
    assert torch.equal(q.scales, scales), (q.scales != scales).nonzero()[:4].tolist()
    whole = (scales != 255).repeat_interleave(16, -1)      # (codes of a NaN block stand for nothing)
    bad = (q.codes != codes) & whole
    assert not bad.any(), (bad.nonzero()[:4].tolist(), q.codes[bad][:4].tolist(), codes[bad][:4].tolist())


def hard_rows(M, K, dtype, gen, dev):
    """Values of all magnitudes, borders between codes among them, zeros, blocks of zeros and of the smallest and largest values."""
    x = torch.randn(M, K, device=dev, generator=gen, dtype=torch.float64)
    x *= torch.exp2(torch.randint(-6, 7, (M, K // 32), device=dev, generator=gen).double()).repeat_interleave(32, 1)
    borders = torch.tensor([0, -0., .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, .5, 4, -.25, -1.75, -5], dtype=torch.float64, device=dev)
    x[0, :16] = borders
    x[-1, -32:-16] = borders * 2.0 ** -9
    x[-1, -1] = 7.75 * 2.0 ** -9
    if M > 1:
        x[1, :32] = 0.0
        x[1, 32:64] = 0.0
        x[1, 40] = torch.finfo(dtype).smallest_normal / 8 if dtype != torch.bfloat16 else 2.0 ** -130
        x[M // 2, -32:] = torch.finfo(dtype).max * torch.linspace(-1, 1, 32, device=dev)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,K", [(1, 32), (1, 64), (3, 96), (2, 2048), (7, 1056), (37, 1408), (130, 4128), (1025, 64), (5, 14336)])
def test_quantize_and_back(cuda, M, K, dtype):
    from promoe_amd import ops
    print(f"case quantize M={M} K={K} {dtype}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(M + K)
    for gap in (0, 16):
        x = rows((M, K), 0.0, dtype, gen, cuda, gap)
        x.copy_(hard_rows(M, max(K, 64), dtype, gen, cuda)[:, :K])
        q = ops.quantize_mx4(x)
        assert q.shape == (M, K) and q.codes.shape == (M, K // 2) and q.scales.shape == (M, K // 32)
        same(q, x)
        v = values(q.codes, q.scales)
        for back in TYPES:
            y = ops.dequantize_mx4(q, back)
            assert y.dtype == back and torch.equal(y.double(), v.to(back).double()), back


def test_quantize_infinities_nan_and_three_dimensions(cuda):
    from promoe_amd import ops
    print("case quantize_nan", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(3)
    for dtype in TYPES:
        x = torch.randn(3, 5, 160, device=cuda, generator=gen).to(dtype)
        x[0, 0, 3], x[1, 4, 159], x[2, 2, 64] = float("nan"), float("inf"), float("-inf")
        q = ops.quantize_mx4(x)
        assert q.shape == (3, 5, 160)
        same(q, x)
        y = ops.dequantize_mx4(q, dtype)
        bad = torch.zeros(3, 5, 5, dtype=torch.bool, device=cuda)
        bad[0, 0, 0] = bad[1, 4, 4] = bad[2, 2, 2] = True
        assert torch.equal(torch.isnan(y), bad.repeat_interleave(32, -1))


def test_quantize_many_rows_past_32_bits_of_offsets(cuda):
    """2.2e9 values in one call: offsets of values pass 2^32 bytes, their number 2^31.  Rows of zeros have zeros for codes."""
    from promoe_amd import ops
    print("case quantize_large", flush=True)
    M, K = 1 << 20, 2112
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)
    at = torch.tensor([0, 1, M // 2, M - 2, M - 1], device=cuda)
    x[at] = torch.randn(5, K, device=cuda, generator=gen).to(torch.bfloat16)
    q = ops.quantize_mx4(x)
    codes, scales = quantised(x[at])
    assert torch.equal(q.codes[at], codes) and torch.equal(q.scales[at], scales)
    assert int((q.codes != 0).any(1).sum()) == 5
    y = ops.dequantize_mx4(q)
    assert torch.equal(y[at].double(), values(codes, scales)) and int((y != 0).any(1).sum()) == 5


def matrix(shape, gen, dev, spread=3):
    """An Mx4 of random codes, its scales over a few powers of two around 1 / sqrt K"""
    from promoe_amd import ops
    *lead, N, K = shape
    codes = torch.randint(0, 256, (*lead, N, K // 2), device=dev, generator=gen, dtype=torch.uint8)
    mid = 126 - (K.bit_length() // 2)
    scales = torch.randint(mid - spread, mid + 1, (*lead, N, K // 32), device=dev, generator=gen, dtype=torch.uint8)
    return ops.Mx4(codes, scales)


def spaced(q, gap, dev):
    """The same values with rows of codes further apart, other codes between them and NaN wherever a block of scales belongs to no row or
    column."""
    from promoe_amd import ops
    *lead, N, K = q.shape
    codes = torch.full((*lead, N + 1, K // 2 + 16 * gap), 0x77, dtype=torch.uint8, device=dev)[..., :N, : K // 2]
    codes.copy_(q.codes)
    s = ops.Mx4(codes, q.scales)
    assert s.codes.data_ptr() == codes.data_ptr()
    rows = torch.nn.functional.pad(q.scales, (0, -(K // 32) % 8, 0, -N % 32), value=255)
    s.blocks.copy_(rows.unflatten(-1, (-1, 8)).unflatten(-3, (-1, 32)).transpose(-3, -2))
    assert torch.equal(s.scales, q.scales)
    return s


def half64(x, w, b, act):
    v = torch.mm(x, w.t().contiguous())
    e = (x.shape[1] / 4 + 40) * 2.0 ** -23 * (1 + 2.0 ** -7) * torch.mm(x.abs(), w.abs().t().contiguous())
    if b is not None:
        v = v + b
        e = e + 2.0 ** -23 * v.abs()
    return v, e, act64(act, v), slope(act, v) * e + (8 + v.abs()) * 2.0 ** -23 * v.abs()


def expect(x, mats, biases, act, residual=None):
    """(value, error before the rounding) for values x and matrices in 64 bits"""
    d = lambda t: None if t is None else t.double()
    _, _, y, e = half64(x, mats[0], d(biases[0]), act)
    if len(mats) == 2:
        u, eu, _, _ = half64(x, mats[1], d(biases[1]), "none")
        y, e = y * u, e * u.abs() + eu * y.abs() + e * eu + 2.0 ** -23 * (y * u).abs()
    if residual is not None:
        y = y + residual.double()
        e = e + 2.0 ** -23 * y.abs()
    return y, e


def product(dev, M, N, K, kind, dtype, act, bias, residual, gated, out_dtype=None, gap=0, seed=0):
    from promoe_amd import ops
    print(f"case mx4 M={M} N={N} K={K} x={kind} {dtype} act={act} bias={bias} res={residual} gated={gated} out={out_dtype} gap={gap}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(seed + 7 * M + N + K)
    x = rows((M, K), 1.0, dtype, gen, dev, 8 * gap)
    xv = x.double()
    if kind == "mx4":
        x = ops.quantize_mx4(x)
        xv = values(x.codes, x.scales)
        x = spaced(x, gap, dev)
    n = 2 if gated else 1
    mats = [spaced(matrix((N, K), gen, dev), gap, dev) for _ in range(n)]
    bs = [rows((1, N), 0.5, dtype, gen, dev)[0] if bias else None for _ in range(n)]
    res = rows((M, N), 1.0, dtype, gen, dev, gap) if residual else None
    out = torch.full((M + 1, N + 3), 7.0, dtype=out_dtype or dtype, device=dev)
    if gated:
        ops.linear_gated_mx4(x, *mats, *bs, act=act, out=out[:M, :N])
    else:
        ops.linear_mx4(x, mats[0], bs[0], act=act, residual=res, out=out[:M, :N])
    torch.cuda.synchronize()
    y, e = expect(xv, [values(m.codes, m.scales) for m in mats], bs, act, res)
    check(out[:M, :N], y, e)
    assert torch.all(out[M:] == 7.0) and torch.all(out[:, N:] == 7.0)


SHAPES = [(1, 1, 32), (1, 17, 96), (1, 2048, 1056), (2, 33, 64), (5, 130, 544), (8, 64, 4096), (9, 65, 288), (16, 48, 1408), (17, 257, 160),
          (24, 512, 512), (31, 100, 992), (33, 31, 32), (48, 96, 2080), (63, 127, 64), (64, 128, 128), (65, 129, 224), (100, 320, 1536),
          (127, 1, 512), (128, 256, 256), (129, 255, 96), (200, 1000, 352), (256, 256, 256), (257, 513, 1056), (300, 96, 4128),
          (511, 640, 192), (1000, 1409, 544), (2049, 300, 96)]


@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_mx4(cuda, M, N, K, dtype, kind):
    i = SHAPES.index((M, N, K))
    product(cuda, M, N, K, kind, dtype, ACTS[i % 6], i % 2 == 0, i % 3 != 1, False, gap=i % 3)


@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_gated_mx4(cuda, M, N, K, dtype, kind):
    i = SHAPES.index((M, N, K))
    product(cuda, M, N, K, kind, dtype, ACTS[(i + 1) % 6], i % 2 == 1, False, True, gap=i % 2)


@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_every_activation_and_fp32_results(cuda, M, act, kind):
    product(cuda, M, 200, 288, kind, torch.bfloat16, act, True, True, False, torch.float32)
    product(cuda, M, 200, 288, kind, torch.float16, act, True, False, True, torch.float32)


@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("M,N,K,gated", [(1, 2048, 10944, False), (1, 10944, 2048, True), (4, 8192, 8192, False), (300, 2048, 10944, False),
                                         (129, 4096, 4096, True), (2000, 4096, 2048, False), (1024, 2816, 2048, True), (4096, 2050, 1056, False),
                                         (77, 16384, 1024, True), (1300, 4099, 2080, False), (700, 2049, 4128, True)])
def test_sizes_of_dense_layers(cuda, M, N, K, gated, kind):
    product(cuda, M, N, K, kind, torch.bfloat16, "silu" if gated else "none", N % 2 == 1, not gated, gated)


# Every tile on sizes that end inside it, with K whole and in pieces.
@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("M,N,K,gated", [(24, 2050, 10944, False), (40, 4099, 14336, False), (100, 4094, 14336, False), (260, 2049, 10944, True),
                                         (500, 2051, 10944, False), (300, 5003, 4128, False), (1000, 2049, 10944, False), (2000, 4097, 2080, True),
                                         (4100, 4099, 1056, False), (900, 1409, 2080, True), (4000, 1409, 544, False), (3000, 700, 8192, False),
                                         (1500, 8190, 544, False), (200, 14330, 1056, True), (600, 10941, 2048, False), (2050, 10941, 1056, False),
                                         (1030, 8203, 4128, False), (2000, 4099, 4128, True), (60, 30, 9984, False)])
def test_every_tile_on_ragged_sizes(cuda, M, N, K, gated, kind):
    f16 = N % 2 == 0
    product(cuda, M, N, K, kind, torch.float16 if f16 else torch.bfloat16, "gelu" if gated else "relu2", True, not gated, gated, gap=1,
            out_dtype=torch.float32 if M % 100 else None)


@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("M,N,K", [(1, 64, 512), (12, 80, 288), (30, 80, 288), (40, 130, 9984), (300, 300, 512)])
def test_residual_in_place_and_aligned_only_to_its_type(cuda, M, N, K, kind):
    """out is the residual; rows of an odd number of elements from an odd offset on."""
    from promoe_amd import ops
    print(f"case mx4_in_place M={M} N={N} K={K} {kind}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(M)
    x, w = rows((M, K), 1.0, torch.bfloat16, gen, cuda), matrix((N, K), gen, cuda)
    xv = x.double()
    if kind == "mx4":
        x = ops.quantize_mx4(x)
        xv = values(x.codes, x.scales)
    buf = torch.randn(1 + M * (N + 5), device=cuda, generator=gen).to(torch.bfloat16)
    res = buf[1:].view(M, N + 5)[:, :N]
    before = buf.clone()
    y, e = expect(xv, [values(w.codes, w.scales)], [None], "none", res)
    assert ops.linear_mx4(x, w, residual=res, out=res) is res
    torch.cuda.synchronize()
    check(res, y, e)
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[1:].view(M, N + 5)[:, :N] = False
    assert torch.equal(buf[keep], before[keep])


@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("M,N,K,gated", [(5, 1100, 512, False), (450, 1100, 288, False), (1000, 1100, 544, True), (1050, 2050, 4128, False)])
def test_rows_far_apart(cuda, M, N, K, gated, kind):
    """Rows nearly 4 MiB apart, so that offsets pass 2^32 bytes: the same bits as from rows side by side."""
    from promoe_amd import ops
    print(f"case mx4_far M={M} N={N} K={K} gated={gated} {kind}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(M)
    ld = (1 << 22) - 16

    def far(t):
        size = t.element_size()
        v = torch.empty((t.shape[0] - 1) * (ld // size) + t.shape[1], dtype=t.dtype, device=cuda).as_strided(t.shape, (ld // size, 1))
        v.copy_(t)
        return v

    x = rows((M, K), 1.0, torch.bfloat16, gen, cuda).contiguous()
    ws = [matrix((N, K), gen, cuda) for _ in range(2 if gated else 1)]
    res = None if gated else rows((M, N), 1.0, torch.bfloat16, gen, cuda).contiguous()
    xq = ops.quantize_mx4(x)
    assert torch.equal(ops.quantize_mx4(far(x)).codes, xq.codes)
    fx, fres = (ops.Mx4(far(xq.codes), xq.scales) if kind == "mx4" else far(x)), None if gated else far(res)
    fw = [ops.Mx4(far(m.codes), m.scales) for m in ws]
    assert torch.equal(ops.dequantize_mx4(fw[0]), ops.dequantize_mx4(ws[0]))
    x = xq if kind == "mx4" else x
    out = torch.empty((M - 1) * (ld // 2) + N, dtype=torch.bfloat16, device=cuda).as_strided((M, N), (ld // 2, 1))
    if gated:
        want = ops.linear_gated_mx4(x, *ws)
        ops.linear_gated_mx4(fx, *fw, out=out)
    else:
        want = ops.linear_mx4(x, ws[0], residual=res)
        ops.linear_mx4(fx, fw[0], residual=fres, out=out)
    assert torch.equal(out, want)


@pytest.mark.parametrize("M", [1, 12, 40, 300])
def test_nan_and_infinities_stay_in_their_rows_and_columns(cuda, M):
    from promoe_amd import ops
    print(f"case mx4_nan M={M}", flush=True)
    N, K = 300, 288
    gen = torch.Generator(device=cuda).manual_seed(M)
    x = rows((M, K), 1.0, torch.float16, gen, cuda)
    w = matrix((N, K), gen, cuda)
    scales = w.scales
    scales[17, 5] = 255
    scales[N - 1, K // 32 - 1] = 255
    w = ops.Mx4(w.codes, scales)
    if M > 1:
        x[M - 1, K - 1] = float("nan")
        x[0, 0] = float("inf")
    wv = values(w.codes, w.scales)
    for t in (torch.float16, torch.bfloat16):
        got = ops.linear_mx4(x.to(t), w).double()
        ref = torch.mm(x.to(t).double(), wv.t().contiguous())
        # (0 of w times infinity is NaN in both)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isposinf(got), torch.isposinf(ref))
    got = ops.linear_mx4(ops.quantize_mx4(x), w)
    bad = torch.zeros(M, N, dtype=torch.bool, device=cuda)
    bad[:, [17, N - 1]] = True
    if M > 1:
        bad[[0, M - 1]] = True
    assert torch.equal(torch.isnan(got), bad)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_scales_of_the_whole_range(cuda, M):
    """Weights around 2^-100 and 2^100 in one matrix, rows the other way: nothing is lost to a narrower type between."""
    from promoe_amd import ops
    print(f"case mx4_scales M={M}", flush=True)
    N, K = 130, 512
    gen = torch.Generator(device=cuda).manual_seed(M)
    codes = matrix((N, K), gen, cuda).codes
    s = torch.full((N, K // 32), 127, dtype=torch.uint8, device=cuda)
    s[0::3] = 27
    s[1::3] = 217
    w = ops.Mx4(codes, s)
    x = rows((M, K), 1.0, torch.bfloat16, gen, cuda)
    x[::2] *= 2.0 ** -20
    for t in (torch.bfloat16, torch.float16):
        for q in (False, True):
            xs = x.to(t)
            xv = xs.double()
            if q:
                xs = ops.quantize_mx4(xs)
                xv = values(xs.codes, xs.scales)
            y, e = expect(xv, [values(codes, s)], [None], "none")
            check(ops.linear_mx4(xs, w, out_dtype=torch.float32), y, e)


@pytest.mark.parametrize("M", [1, 12, 40, 300])
def test_fp16_rows_at_the_ends_of_what_fp16_weights_can_be(cuda, M):
    """Scales of 2^-23 and 2^13 (the last whose codes are all fp16), one step further, and rows of the smallest fp16 values."""
    from promoe_amd import ops
    print(f"case mx4_fp16 M={M}", flush=True)
    N, K = 200, 1056
    gen = torch.Generator(device=cuda).manual_seed(M)
    codes = matrix((N, K), gen, cuda).codes
    x = rows((M, K), 1.0, torch.float16, gen, cuda)
    x[::2] *= 2.0 ** -22
    for low, high in ((104, 105), (139, 140), (103, 105), (139, 141), (104, 140), (127, 128)):
        s = torch.randint(low, high + 1, (N, K // 32), device=cuda, generator=gen, dtype=torch.uint8)
        w = ops.Mx4(codes, s)
        y, e = expect(x.double(), [values(codes, s)], [None], "none")
        check(ops.linear_mx4(x, w, out_dtype=torch.float32), y, e)
        y, e = expect(x.double(), [values(codes, s)] * 2, [None] * 2, "relu")
        check(ops.linear_gated_mx4(x, w, w, act="relu", out_dtype=torch.float32), y, e)


def routed(T, E, k, gen, dev, skew=0.0, left=0.0):
    from promoe_amd import ops
    s = torch.randn(T, E, device=dev, generator=gen) - skew * torch.log1p(torch.arange(E, device=dev))
    idx = torch.topk(s, k, dim=1).indices.int() if T else torch.empty(0, k, dtype=torch.int32, device=dev)
    if left:
        idx[torch.rand(T, k, device=dev, generator=gen) < left] = -1
    return idx, ops.dispatch(idx.contiguous(), E)


def experts(dev, T, E, k, N, K, kind, dtype, gated, of_tokens, bias=False, act="silu", out_dtype=None, gap=0, skew=0.0, left=0.0):
    from promoe_amd import ops
    print(f"case mx4_experts T={T} E={E} k={k} N={N} K={K} x={kind} {dtype} gated={gated} tokens={of_tokens} gap={gap} skew={skew} left={left}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(7 * T + N + K)
    idx, d = routed(T, E, k, gen, dev, skew, left)
    P = T * k
    x = rows((T if of_tokens else P, K), 1.0, dtype, gen, dev, 8 * gap)
    xv = x.double()
    if kind == "mx4":
        x = ops.quantize_mx4(x)
        xv = values(x.codes, x.scales)
        x = spaced(x, gap, dev)
    n = 2 if gated else 1
    mats = [spaced(matrix((E, N, K), gen, dev), gap, dev) for _ in range(n)]
    bs = [rows((E, N), 0.5, dtype, gen, dev).contiguous() if bias else None for _ in range(n)]
    out = torch.full((P + 1, N + 3), 7.0, dtype=out_dtype or dtype, device=dev)
    call = ops.experts_gated_mx4 if gated else ops.experts_linear_mx4
    a = act if gated else "none"
    call(x, *mats, d, *bs, act=a, of_tokens=of_tokens, out=out[:P, :N])
    torch.cuda.synchronize()
    flat = idx.reshape(-1).cpu()
    at = 0
    for e in range(E):
        pairs = torch.nonzero(flat == e)[:, 0].to(dev)
        if pairs.numel():
            src = xv[pairs // k] if of_tokens else xv[at: at + pairs.numel()]
            y, err = expect(src, [values(m.codes[e], m.scales[e]) for m in mats], [b if b is None else b[e] for b in bs], a)
            check(out[at: at + pairs.numel(), :N], y, err)
        at += pairs.numel()
    assert torch.all(out[at:] == 7.0) and torch.all(out[:, N:] == 7.0)


EXPERTS = [(1, 8, 1, 33, 32), (1, 64, 6, 128, 256), (2, 8, 2, 130, 544), (5, 60, 4, 65, 1408), (33, 64, 8, 100, 96), (64, 16, 1, 257, 160),
           (100, 256, 8, 48, 64), (130, 8, 2, 320, 1056), (379, 60, 4, 129, 288), (700, 8, 8, 96, 512), (1500, 64, 6, 255, 256), (2000, 4, 2, 513, 288)]


@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("gated", [False, True], ids=["linear", "gated"])
@pytest.mark.parametrize("T,E,k,N,K", EXPERTS)
def test_experts(cuda, T, E, k, N, K, gated, kind):
    i = EXPERTS.index((T, E, k, N, K))
    experts(cuda, T, E, k, N, K, kind, [torch.bfloat16, torch.float16][i % 2], gated, gated, i % 3 == 0, ["silu", "gelu", "gelu_tanh"][i % 3],
            torch.float32 if i % 4 == 3 else None, gap=i % 2, skew=[0.0, 3.0][i % 2], left=[0.0, 0.0, 0.3][i % 3])


@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("T,E,k,N,K,gated,skew", [(900, 700, 3, 130, 288, True, 0.0), (6000, 700, 3, 70, 288, False, 1.0), (3000, 256, 4, 100, 544, True, 2.0),
                                                  (300, 8, 2, 1000, 2080, False, 0.0), (1100, 8, 2, 1050, 1056, True, 1.0), (5000, 16, 2, 513, 544, False, 0.5),
                                                  (2000, 64, 1, 260, 96, True, 4.0), (200, 64, 1, 100, 288, False, 20.0)])
def test_many_experts_and_uneven_ones(cuda, T, E, k, N, K, gated, skew, kind):
    """More experts than lanes, single rows behind whole tiles, most rows at a few experts."""
    experts(cuda, T, E, k, N, K, kind, torch.float16 if T % 3 else torch.bfloat16, gated, gated, bias=True, gap=1, skew=skew)


@pytest.mark.parametrize("kind", ["mx4", "16"])
@pytest.mark.parametrize("T,E,k,N,K,gated", [(1, 64, 6, 1408, 2048, True), (1, 64, 6, 2048, 1408, False), (20, 64, 8, 3584, 2560, False),
                                             (300, 64, 6, 1408, 2048, True), (1024, 8, 2, 4096, 2048, False)])
def test_sizes_of_experts(cuda, T, E, k, N, K, gated, kind):
    experts(cuda, T, E, k, N, K, kind, torch.bfloat16, gated, gated)


def test_more_rows_of_tokens_or_of_experts_than_the_other(cuda):
    """of_tokens with the second half's shape and rows in order with the first half's: both ways of reading x for both products."""
    for kind in ("mx4", "16"):
        experts(cuda, 50, 8, 3, 70, 96, kind, torch.bfloat16, False, True)
        experts(cuda, 50, 8, 3, 70, 96, kind, torch.bfloat16, True, False)
        experts(cuda, 400, 8, 3, 200, 160, kind, torch.bfloat16, False, True)
        experts(cuda, 400, 8, 3, 200, 160, kind, torch.bfloat16, True, False)


def test_one_expert_has_all_rows_and_none_has_any(cuda):
    from promoe_amd import ops
    print("case mx4_one_expert", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(2)
    for T in (3, 300):
        x = rows((T, 96), 1.0, torch.bfloat16, gen, cuda).contiguous()
        w = matrix((9, 70, 96), gen, cuda)
        d = ops.dispatch(torch.full((T, 1), 8, dtype=torch.int32, device=cuda), 9)
        y, e = expect(x.double(), [values(w.codes[8], w.scales[8])], [None], "none")
        check(ops.experts_linear_mx4(x, w, d), y, e)
        d = ops.dispatch(torch.full((T, 1), -1, dtype=torch.int32, device=cuda), 9)
        out = torch.full((T, 70), 7.0, dtype=torch.bfloat16, device=cuda)
        assert torch.all(ops.experts_linear_mx4(x, w, d, out=out) == 7.0)


def layer(x, wg, wu, wd, E, k, logits, quantise):
    """A sparse block: routing, both halves of the experts, the way back"""
    from promoe_amd import ops
    idx, w = ops.topk(logits, k, 1)
    d = ops.dispatch(idx, E)
    q = ops.quantize_mx4 if quantise else (lambda t: t)
    h = ops.experts_gated_mx4(q(x), wg, wu, d, of_tokens=True, out_dtype=torch.bfloat16)
    return idx, w, ops.unsort_tokens(ops.experts_linear_mx4(q(h), wd, d, out_dtype=torch.bfloat16), d, w), h, d


@pytest.mark.parametrize("quantise", [False, True], ids=["16", "mx4"])
@pytest.mark.parametrize("T", [1, 7, 40, 500])
def test_a_sparse_block(cuda, T, quantise):
    """Both halves and the way back against 64 bits from the rows between the halves on (their rounding is part of the block)."""
    print(f"case mx4_block T={T} {quantise}", flush=True)
    E, k, H, I = 16, 4, 256, 192
    gen = torch.Generator(device=cuda).manual_seed(T)
    x = torch.randn(T, H, device=cuda, generator=gen).to(torch.bfloat16)
    wg, wu, wd = matrix((E, I, H), gen, cuda), matrix((E, I, H), gen, cuda), matrix((E, H, I), gen, cuda)
    logits = torch.randn(T, E, device=cuda, generator=gen)
    idx, w, y, h, d = layer(x, wg, wu, wd, E, k, logits, quantise)
    torch.cuda.synchronize()

    def form(t):
        return values(*quantised(t)) if quantise else t.double()

    order = torch.sort(idx.reshape(-1), stable=True).indices
    which = idx.reshape(-1)[order].long()
    ref, err = torch.zeros(T, H, dtype=torch.float64, device=cuda), torch.zeros(T, H, dtype=torch.float64, device=cuda)
    for e in range(E):
        at = torch.nonzero(which == e)[:, 0]
        if at.numel():
            hy, he = expect(form(x)[order[at] // k], [values(m.codes[e], m.scales[e]) for m in (wg, wu)], [None, None], "silu")
            check(h[at], hy, he)
            v, ve = expect(form(h)[at], [values(wd.codes[e], wd.scales[e])], [None], "none")
            ve = ve * (1 + 2.0 ** -8) + 2.0 ** -8 * (v.abs() + ve)              # the product's rows are bf16
            ww = w.double().reshape(-1)[order[at], None]
            ref.index_add_(0, order[at] // k, v * ww)
            err.index_add_(0, order[at] // k, (ve + 2.0 ** -22 * v.abs()) * ww)
    check(y, ref, err)


def test_empty_other_stream_graphs_and_refusals(cuda):
    from promoe_amd import _lib as L
    from promoe_amd import ops
    print("case mx4_graph", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(5)
    bf = dict(dtype=torch.bfloat16, device=cuda)
    E, k, H, I = 8, 2, 256, 352
    wg, wu, wd = matrix((E, I, H), gen, cuda), matrix((E, I, H), gen, cuda), matrix((E, H, I), gen, cuda)
    w2 = matrix((I, H), gen, cuda)
    assert ops.linear_mx4(torch.empty(0, H, **bf), w2).shape == (0, I)
    assert ops.linear_mx4(ops.quantize_mx4(torch.empty(0, H, **bf)), w2).shape == (0, I)
    assert ops.dequantize_mx4(ops.quantize_mx4(torch.empty(0, H, **bf))).shape == (0, H)
    st = torch.cuda.Stream()
    for T in (1, 30, 400):
        x, logits = torch.randn(T, H, device=cuda, generator=gen).to(torch.bfloat16), torch.randn(T, E, device=cuda, generator=gen)
        for quantise in (False, True):
            q = ops.quantize_mx4 if quantise else (lambda t: t)
            block = lambda t: layer(t, wg, wu, wd, E, k, logits, quantise)[2] + ops.linear_mx4(q(t), w2, act="silu")[:, :H]
            want = block(x)
            torch.cuda.synchronize()
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                assert torch.equal(block(x), want)
            torch.cuda.synchronize()
            xg = x.clone()
            g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = block(xg)
            with torch.cuda.graph(g2):             # a second graph beside it, each with memory of its own
                y2 = block(xg)
            for i in range(4):
                xg.copy_(x * (1 + i))
                g.replay()
                g2.replay()
                torch.cuda.synchronize()
                want = block(xg)
                assert torch.equal(y, want) and torch.equal(y2, want)
    x = torch.randn(40, H, device=cuda, generator=gen).to(torch.bfloat16)
    d = ops.dispatch(torch.zeros(40, 1, dtype=torch.int32, device=cuda), E)
    xq = ops.quantize_mx4(x)
    cpu = ops.Mx4(w2.codes.cpu(), w2.scales.cpu())
    for call in (lambda: ops.linear_mx4(x.float(), w2), lambda: ops.linear_mx4(x, w2, torch.zeros(I, device=cuda)),
                 lambda: ops.linear_mx4(x[:, :224], w2), lambda: ops.linear_mx4(x, w2, residual=x), lambda: ops.linear_mx4(x, w2.codes),
                 lambda: ops.linear_mx4(x, w2, out=torch.empty(40, I - 1, **bf)), lambda: ops.linear_mx4(x, w2, out_dtype=torch.float16),
                 lambda: ops.linear_mx4(x, cpu), lambda: ops.linear_mx4(x.cpu(), w2), lambda: ops.linear_mx4(x, wg),
                 lambda: ops.linear_mx4(xq, w2, torch.zeros(I, **bf), out_dtype=torch.float16), lambda: ops.linear_gated_mx4(x, w2, matrix((I + 1, H), gen, cuda)),
                 lambda: ops.linear_gated_mx4(x, w2, spaced(w2, 1, cuda)), lambda: ops.experts_linear_mx4(x, w2, d),
                 lambda: ops.experts_linear_mx4(x[:39], wg, d), lambda: ops.experts_linear_mx4(x, matrix((E - 1, I, H), gen, cuda), d),
                 lambda: ops.experts_gated_mx4(x, wg, wu, d, b_gate=torch.zeros(I, **bf)), lambda: ops.quantize_mx4(x[:, :200]),
                 lambda: ops.quantize_mx4(x.double()), lambda: ops.quantize_mx4(x[:, 4:36]), lambda: ops.quantize_mx4(x.cpu()),
                 lambda: ops.quantize_mx4(x.t()), lambda: ops.linear_mx4(x, w2, act="tanh"), lambda: ops.dequantize_mx4(xq, torch.float64),
                 lambda: ops.linear_gated_mx4(x, w2, None), lambda: ops.experts_linear_mx4(x, wg, ops.dispatch(torch.zeros(40, 1, dtype=torch.int32, device=cuda), E, max_units=2))):
        with pytest.raises(L.MoeError):
            call()
    x.requires_grad_(True)
    for call in (lambda: ops.linear_mx4(x, w2), lambda: ops.quantize_mx4(x), lambda: ops.experts_linear_mx4(x, wg, d)):
        with pytest.raises(L.MoeError, match="gradient"):
            call()


def test_two_streams_at_once(cuda):
    """Two calls of different inputs on two streams, many times: nothing is shared between calls."""
    from promoe_amd import ops
    print("case mx4_two_streams", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(8)
    w = matrix((700, 1056), gen, cuda)
    xs = [torch.randn(M, 1056, device=cuda, generator=gen).to(torch.bfloat16) for M in (100, 300)]
    want = [ops.linear_mx4(ops.quantize_mx4(x), w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.linear_mx4(ops.quantize_mx4(xs[i]), w))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_matrices_as_they_come(cuda):
    """Scales in any order, codes off 16-byte boundaries (copied) or far apart (kept), parts of stacked matrices, matrices from quantize_mx4."""
    from promoe_amd import ops
    print("case mx4_layouts", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(6)
    N, K = 37, 96
    q = matrix((N, K), gen, cuda)
    v = values(q.codes, q.scales)
    off = torch.empty(N * 48 + 8, dtype=torch.uint8, device=cuda)[8:].view(N, 48)
    off.copy_(q.codes)
    x = torch.randn(50, K, device=cuda, generator=gen).to(torch.bfloat16)
    y, e = expect(x.double(), [v], [None], "none")
    for codes, scales in ((off, q.scales), (off.t().contiguous().t(), q.scales.t().contiguous().t())):
        m = ops.Mx4(codes, scales)
        assert torch.equal(m.codes, q.codes) and torch.equal(m.scales, q.scales)
        check(ops.linear_mx4(x, m), y, e)
        assert torch.equal(ops.dequantize_mx4(m, torch.float32).double(), v)
    three = matrix((3, N, K), gen, cuda)
    part = ops.Mx4(three.codes[:, 5:30], three.scales[:, 5:30])
    assert part.codes.data_ptr() == three.codes[:, 5:30].data_ptr()
    assert torch.equal(ops.dequantize_mx4(part, torch.float32).double(), values(three.codes[:, 5:30], three.scales[:, 5:30]))
    # a pair, one quantised here and one given as codes and scales
    w = ops.quantize_mx4(torch.randn(N, K, device=cuda, generator=gen))
    y, e = expect(x.double(), [values(w.codes, w.scales), v], [None, None], "silu")
    check(ops.linear_gated_mx4(x, w, q), y, e)
    # matrices of experts quantised from rows that lie apart
    src = torch.randn(4, N + 3, 2 * K, device=cuda, generator=gen)[:, :N, :K]
    w = ops.quantize_mx4(src)
    same(w, src)
    idx, d = routed(50, 4, 2, gen, cuda)
    got = ops.experts_linear_mx4(x, w, d, of_tokens=True, out_dtype=torch.float32)
    order = torch.sort(idx.reshape(-1), stable=True).indices
    for e_ in range(4):
        at = torch.nonzero(idx.reshape(-1)[order] == e_)[:, 0]
        y, e = expect(x.double()[order[at] // 2], [values(w.codes[e_], w.scales[e_])], [None], "none")
        check(got[at], y, e)
