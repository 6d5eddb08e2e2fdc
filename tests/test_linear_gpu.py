"""Dense products on the GPU against the same formula in 64 bits.

Tolerance of an element.  A product of two 16-bit values is exact in fp32.  The sum of K of them goes through blocks of at least 8 in
the matrix core and then at most K / 8 + 8 additions, each of which rounds (or cuts) by at most 2^-23 of what is added up so far:
e = (K / 8 + 40) 2^-23 sum |x w| (40: the blocks' own steps, the bias and the join of partial sums).  An activation with slope s
passes on s e, and its own arithmetic (2^x, reciprocal, erfc: a few units, the exponent off by |v| 2^-24) adds (8 + |v|) 2^-23 |v|.  A gated
product adds the terms of both factors.  The rounding to the result's type is half a step: 2^-8 (bf16), 2^-11 (fp16) of the value,
2^-24 for fp32, and half of the smallest step of fp16 (2^-25) near zero."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
ACTS = ["none", "silu", "gelu", "gelu_tanh", "relu", "relu2"]


def act64(name, v):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return v * torch.special.erfc(-v / math.sqrt(2)) / 2
    if name == "gelu_tanh":
        return v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))) / 2
    return {"none": v, "relu": v.clamp(min=0), "relu2": v.clamp(min=0) ** 2}[name]


def slope(name, v):
    return 2 * v.abs() + 1e-3 if name == "relu2" else 1.0 if name in ("none", "relu") else 1.13


def half64(x, w, b, act):
    v = torch.mm(x, w.t().contiguous())
    e = (x.shape[1] / 8 + 40) * 2.0 ** -23 * torch.mm(x.abs(), w.abs().t().contiguous())
    if b is not None:
        v = v + b
        e = e + 2.0 ** -23 * v.abs()
    return v, e, act64(act, v), slope(act, v) * e + (8 + v.abs()) * 2.0 ** -23 * v.abs()


def expect(x, mats, biases, act, residual):
    """(value, error before the rounding) in 64 bits"""
    d = lambda t: None if t is None else t.double()
    x = x.double()
    _, _, y, e = half64(x, mats[0].double(), d(biases[0]), act)
    if len(mats) == 2:
        u, eu, _, _ = half64(x, mats[1].double(), d(biases[1]), "none")
        y, e = y * u, e * u.abs() + eu * y.abs() + e * eu + 2.0 ** -23 * (y * u).abs()
    if residual is not None:
        y = y + residual.double()
        e = e + 2.0 ** -23 * y.abs()
    return y, e


def check(got, y, e):
    tol = e * (1 + 2.0 ** -8) + HALF[got.dtype] * (y.abs() + e) + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -130)
    bad = ~((got.double() - y).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4].tolist(), y[bad][:4].tolist(), tol[bad][:4].tolist(), bad.nonzero()[:4].tolist())


def rows(shape, std, dtype, gen, dev, gap=0, fill=float("nan")):
    """A matrix whose rows lie `gap` elements further apart, with NaN between them and behind the last."""
    t = torch.full((shape[0] + 1, shape[1] + gap), fill, dtype=dtype, device=dev)
    v = t[: shape[0], : shape[1]]
    v.copy_((torch.randn(shape, device=dev, generator=gen) * std).to(dtype))
    return v


def run(dev, M, N, K, dtype, act, bias, residual, gated, out_dtype=None, gap=0, seed=0):
    from promoe_amd import ops
    print(f"case linear M={M} N={N} K={K} {dtype} act={act} bias={bias} res={residual} gated={gated} out={out_dtype} gap={gap}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(seed + 7 * M + N + K)
    x = rows((M, K), 1.0, dtype, gen, dev, gap)
    n = 2 if gated else 1
    mats = [rows((N, K), K ** -0.5, dtype, gen, dev, gap) for _ in range(n)]
    bs = [rows((1, N), 0.5, dtype, gen, dev)[0] if bias else None for _ in range(n)]
    res = rows((M, N), 1.0, dtype, gen, dev, gap) if residual else None
    out = torch.full((M + 1, N + 3), 7.0, dtype=out_dtype or dtype, device=dev)
    kw = dict(act=act, out=out[:M, :N])
    if gated:
        got = ops.linear_gated(x, mats[0], mats[1], bs[0], bs[1], **kw)
    else:
        got = ops.linear(x, mats[0], bs[0], residual=res, **kw)
    torch.cuda.synchronize()
    y, e = expect(x, mats, bs, act, res)
    check(got, y, e)
    assert torch.all(out[M:] == 7.0) and torch.all(out[:, N:] == 7.0)


SHAPES = [(1, 1, 8), (1, 17, 24), (1, 2048, 1032), (2, 33, 72), (5, 130, 520), (8, 64, 4096), (9, 65, 264), (16, 48, 1408), (17, 257, 136),
          (24, 512, 512), (31, 100, 1000), (33, 31, 40), (48, 96, 2056), (63, 127, 64), (64, 128, 128), (65, 129, 200), (100, 320, 1536),
          (127, 1, 512), (128, 256, 64), (129, 255, 56), (200, 1000, 328), (256, 256, 256), (257, 513, 1032), (300, 96, 4104),
          (511, 640, 192), (1000, 1409, 520), (2049, 300, 72)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(cuda, M, N, K, dtype):
    i = SHAPES.index((M, N, K))
    run(cuda, M, N, K, dtype, ACTS[i % 6], i % 2 == 0, i % 3 != 1, False, gap=8 * (i % 3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_gated(cuda, M, N, K, dtype):
    i = SHAPES.index((M, N, K))
    run(cuda, M, N, K, dtype, ACTS[(i + 1) % 6], i % 2 == 1, False, True, gap=8 * (i % 2))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_every_activation_with_everything_else(cuda, M, act):
    run(cuda, M, 200, 264, torch.bfloat16, act, True, True, False)
    run(cuda, M, 200, 264, torch.float16, act, True, False, True)


@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (3, 64, 1408), (40, 500, 264), (130, 257, 1032), (600, 512, 512)])
def test_results_in_fp32(cuda, M, N, K):
    run(cuda, M, N, K, torch.bfloat16, "none", True, True, False, out_dtype=torch.float32)
    run(cuda, M, N, K, torch.float16, "gelu", False, False, False, out_dtype=torch.float32)
    run(cuda, M, N, K, torch.bfloat16, "silu", False, False, True, out_dtype=torch.float32)


@pytest.mark.parametrize("M,N,K,gated", [(1, 2048, 10944, False), (1, 10944, 2048, True), (4, 8192, 8192, False), (300, 2048, 10944, False),
                                         (129, 4096, 4096, True), (2000, 4096, 2048, False), (1024, 2816, 2048, True), (4096, 2050, 1032, False),
                                         (77, 16384, 1024, True)])
def test_sizes_of_dense_layers(cuda, M, N, K, gated):
    run(cuda, M, N, K, torch.bfloat16, "silu" if gated else "none", False, not gated, gated)


@pytest.mark.parametrize("M,N,K,gated", [(1184, 13754, 2112, False), (768, 10944, 2056, True), (4104, 4090, 2056, False), (4120, 2041, 1032, True),
                                         (4090, 8203, 1032, False)])
def test_products_cut_in_two_launches(cuda, M, N, K, gated):
    """Whole rounds of the widest tile, and the columns or rows behind them."""
    run(cuda, M, N, K, torch.bfloat16 if N % 2 else torch.float16, "silu" if gated else "none", True, not gated, gated, gap=8 * (N % 2))
    run(cuda, M, N, K, torch.bfloat16, "none", False, False, gated, out_dtype=torch.float32)


# Every tile on sizes that end inside it, with K whole and in pieces, and more tiles than workgroups of the widest one.
@pytest.mark.parametrize("M,N,K,gated", [(130, 2049, 4104, False), (510, 4093, 4104, False), (450, 4099, 2056, False), (260, 2049, 10952, False), (512, 4099, 1032, False),
                                         (1030, 1023, 8200, False), (1000, 4099, 1032, False), (768, 2050, 10952, False), (2000, 4097, 520, False),
                                         (1300, 2050, 10952, False), (4090, 8203, 1032, False), (100, 320, 1544, True), (1000, 1409, 520, True),
                                         (512, 2051, 4104, True), (1300, 1021, 10952, True), (4090, 4101, 1032, True)])
def test_every_tile_on_ragged_sizes(cuda, M, N, K, gated):
    f16 = N % 2 == 0
    run(cuda, M, N, K, torch.float16 if f16 else torch.bfloat16, "gelu" if gated else "relu2", True, not gated, gated, gap=8,
        out_dtype=torch.float32 if f16 and gated else None)


@pytest.mark.parametrize("M,N,K", [(1, 64, 512), (30, 80, 264), (300, 300, 512)])
def test_residual_in_place_and_aligned_only_to_its_type(cuda, M, N, K):
    """out is the residual; rows of an odd number of elements from an odd offset on."""
    from promoe_amd import ops
    print(f"case linear_in_place M={M} N={N} K={K}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(M)
    x, w = rows((M, K), 1.0, torch.bfloat16, gen, cuda), rows((N, K), K ** -0.5, torch.bfloat16, gen, cuda)
    buf = torch.randn(1 + M * (N + 5), device=cuda, generator=gen).to(torch.bfloat16)
    res = buf[1:].view(M, N + 5)[:, :N]
    before = buf.clone()
    y, e = expect(x, [w], [None], "none", res)
    assert ops.linear(x, w, residual=res, out=res) is res
    torch.cuda.synchronize()
    check(res, y, e)
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[1:].view(M, N + 5)[:, :N] = False
    assert torch.equal(buf[keep], before[keep])


@pytest.mark.parametrize("M", [1, 30, 300])
def test_infinities_and_nan_stay_in_their_rows_and_columns(cuda, M):
    from promoe_amd import ops
    N, K = 300, 264
    print(f"case linear_nan M={M}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(M)
    x, w = rows((M, K), 1.0, torch.float16, gen, cuda), rows((N, K), K ** -0.5, torch.float16, gen, cuda)
    w[17, 5] = float("nan")
    w[N - 1, K - 1] = float("inf")
    if M > 1:
        x[M - 1, K - 1] = float("nan")
        x[0, 0] = float("inf")
    for act in ACTS:
        got = ops.linear(x, w, act=act).float()
        ref = act64(act, torch.mm(x.float(), w.float().t().contiguous()))
        assert torch.equal(torch.isnan(got), torch.isnan(ref)), act
        assert torch.equal(torch.isposinf(got), torch.isposinf(ref)), act


def test_empty_other_stream_graph_and_refusals(cuda):
    from promoe_amd import _lib as L
    from promoe_amd import ops
    print("case linear_graph", flush=True)
    bf = dict(dtype=torch.bfloat16, device=cuda)
    assert ops.linear(torch.empty(0, 64, **bf), torch.empty(32, 64, **bf)).shape == (0, 32)
    assert ops.linear_gated(torch.empty(3, 64, **bf), torch.empty(0, 64, **bf), torch.empty(0, 64, **bf)).shape == (3, 0)
    gen = torch.Generator(device=cuda).manual_seed(5)
    xs = [rows((M, 1408), 1.0, torch.bfloat16, gen, cuda).contiguous() for M in (1, 40, 300)]
    w, u = (rows((512, 1408), 0.03, torch.bfloat16, gen, cuda).contiguous() for _ in range(2))
    down = rows((1408, 512), 0.04, torch.bfloat16, gen, cuda).contiguous()
    layer = lambda x: ops.linear(ops.linear_gated(x, w, u), down, residual=x)
    st = torch.cuda.Stream()
    for x in xs:
        want = layer(x)
        torch.cuda.synchronize()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            assert torch.equal(layer(x), want)
        torch.cuda.synchronize()
        xg = x.clone()
        g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(xg)
        with torch.cuda.graph(g2):                 # a second graph beside it, each with memory of its own
            y2 = layer(xg)
        for i in range(4):
            xg.copy_(x * (1 + i))
            g.replay()
            g2.replay()
            torch.cuda.synchronize()
            want = layer(xg)
            assert torch.equal(y, want) and torch.equal(y2, want)
    x = xs[1]
    for call in (lambda: ops.linear(x, w.half()), lambda: ops.linear(x, w, torch.zeros(512, device=cuda)), lambda: ops.linear(x, w[:, :1400]),
                 lambda: ops.linear(x, w, residual=x), lambda: ops.linear(x, w, out=torch.empty(40, 511, **bf)),
                 lambda: ops.linear(x, w, out_dtype=torch.float16), lambda: ops.linear(x.t(), w), lambda: ops.linear_gated(x, w, u[:511]),
                 lambda: ops.linear(x[:, 4:], w[:, 4:]), lambda: ops.linear(x.cpu(), w), lambda: ops.linear(x[:, :1404], w[:, :1404])):
        with pytest.raises(L.MoeError):
            call()
    w.requires_grad_(True)
    with pytest.raises(L.MoeError, match="gradient"):
        ops.linear(x, w)
    with torch.no_grad():
        ops.linear(x, w)


def test_a_result_beside_its_operand_in_one_buffer(cuda):
    """x and y as columns of one matrix; y over x is refused."""
    from promoe_amd import _lib as L
    from promoe_amd import ops
    print("case linear_beside", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(9)
    for M in (1, 5, 70):
        buf = torch.randn(M, 192, device=cuda, generator=gen).to(torch.bfloat16)
        w = rows((64, 128), 0.1, torch.bfloat16, gen, cuda)
        y, e = expect(buf[:, :128], [w], [None], "none", None)
        check(ops.linear(buf[:, :128], w, out=buf[:, 128:]), y, e)
        for out in (buf[:, 127:191], buf[:, :64]):
            with pytest.raises(L.MoeError, match="overlaps"):
                ops.linear(buf[:, :128], w, out=out)


@pytest.mark.parametrize("M,N,K,gated", [(5, 1100, 512, False), (450, 1100, 264, False), (1000, 1409, 520, True), (2000, 1030, 8200, False)])
def test_rows_far_apart(cuda, M, N, K, gated):
    """Rows 4 MiB apart, so that offsets pass 2^31 elements and 2^32 bytes: the same bits as from rows side by side."""
    from promoe_amd import ops
    print(f"case linear_far M={M} N={N} K={K} gated={gated}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(M)
    ld = (1 << 21) - 8

    def far(t):
        v = torch.empty((t.shape[0] - 1) * ld + t.shape[1], dtype=t.dtype, device=cuda).as_strided(t.shape, (ld, 1))
        v.copy_(t)
        return v

    x, w, u = (rows(s, 0.1, torch.bfloat16, gen, cuda).contiguous() for s in ((M, K), (N, K), (N, K)))
    res = rows((M, N), 1.0, torch.bfloat16, gen, cuda).contiguous()
    out = torch.empty((M - 1) * ld + N, dtype=torch.bfloat16, device=cuda).as_strided((M, N), (ld, 1))
    if gated:
        want = ops.linear_gated(x, w, u)
        ops.linear_gated(far(x), far(w), far(u), out=out)
    else:
        want = ops.linear(x, w, residual=res)
        ops.linear(far(x), far(w), residual=far(res), out=out)
    assert torch.equal(out, want)
