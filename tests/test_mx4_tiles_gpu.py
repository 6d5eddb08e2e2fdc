"""Every kernel that a product in 4 bits can take, on sizes that end inside its tiles.

CASES has one product for each kind of x, single or gated, dense or by expert, tile, number of slabs in LDS, K whole or in pieces; that it has
them all is checked on the CPU against what the plan gives over the whole range of sizes.  Tolerances: test_mx4_gpu.py."""
import ctypes
import math
import random

import pytest
import torch

from tests.test_linear_gpu import ACTS, check, rows
from tests.test_mx4_gpu import expect, matrix, spaced, values

# x in 4 or 16 bits, gated, (experts, choices) or dense, rows (by expert: tokens), N, K
CASES = [
    ("16", False, None, 1, 61, 96), ("16", False, None, 17, 61, 96), ("16", False, None, 17, 63, 2496), ("16", False, None, 6703, 277, 96),
    ("16", False, None, 8911, 65, 4032), ("16", False, None, 8408, 193, 96), ("16", False, None, 9251, 197, 5600), ("16", False, None, 8734, 193, 544),
    ("16", False, None, 8240, 65, 3872), ("16", False, None, 8318, 459, 1056), ("16", False, None, 5677, 129, 10112),
    ("16", False, (2, 2), 3, 61, 96), ("16", False, (2, 1), 46, 61, 96), ("16", False, (8, 4), 4135, 69, 96), ("16", False, (8, 3), 2667, 203, 96),
    ("16", False, (3, 3), 6660, 69, 800), ("16", False, (4, 2), 5562, 405, 1568),
    ("16", True, None, 1, 61, 96), ("16", True, None, 18, 61, 96), ("16", True, None, 18, 61, 1728), ("16", True, None, 8345, 65, 96),
    ("16", True, None, 9570, 65, 4160), ("16", True, None, 8470, 65, 544), ("16", True, None, 2753, 65, 3616), ("16", True, None, 8461, 197, 1056),
    ("16", True, None, 8237, 65, 5760),
    ("16", True, (2, 1), 4, 61, 96), ("16", True, (2, 1), 36, 65, 96), ("16", True, (4, 3), 2728, 65, 96), ("16", True, (8, 1), 8007, 65, 544),
    ("16", True, (3, 2), 11133, 69, 1568),
    ("mx4", False, None, 1, 61, 96), ("mx4", False, None, 9, 61, 288), ("mx4", False, None, 10, 61, 8576), ("mx4", False, None, 9, 61, 96),
    ("mx4", False, None, 9, 5617, 15648), ("mx4", False, None, 8373, 73, 800), ("mx4", False, None, 2784, 71, 15040), ("mx4", False, None, 8472, 423, 96),
    ("mx4", False, None, 8282, 215, 1120), ("mx4", False, None, 8485, 65, 11200), ("mx4", False, None, 8217, 413, 1568), ("mx4", False, None, 7332, 1047, 96),
    ("mx4", False, None, 9633, 399, 14816),
    ("mx4", False, (2, 1), 7, 61, 96), ("mx4", False, (2, 2), 10, 63, 288), ("mx4", False, (2, 2), 10, 61, 96), ("mx4", False, (2, 1), 8273, 69, 800),
    ("mx4", False, (3, 3), 11783, 67, 96), ("mx4", False, (2, 2), 8279, 81, 1056), ("mx4", False, (8, 3), 6801, 133, 2112), ("mx4", False, (4, 4), 11249, 131, 96),
    ("mx4", True, None, 1, 61, 96), ("mx4", True, None, 10, 61, 96), ("mx4", True, None, 10, 61, 5184), ("mx4", True, None, 10, 61, 800),
    ("mx4", True, None, 9, 61, 4960), ("mx4", True, None, 8359, 197, 96), ("mx4", True, None, 6877, 1, 8096), ("mx4", True, None, 8381, 67, 1312),
    ("mx4", True, None, 2878, 67, 9856), ("mx4", True, None, 8655, 205, 1568), ("mx4", True, None, 8204, 67, 14208), ("mx4", True, None, 8227, 469, 96),
    ("mx4", True, None, 8531, 197, 12064),
    ("mx4", True, (2, 1), 8, 61, 96), ("mx4", True, (2, 2), 10, 63, 96), ("mx4", True, (2, 2), 13, 67, 800), ("mx4", True, (4, 2), 9173, 69, 96),
    ("mx4", True, (4, 1), 8849, 71, 1312), ("mx4", True, (8, 3), 10785, 85, 544), ("mx4", True, (64, 4), 9891, 65, 96),
]
# more than one column of tiles as well
WIDER = [("mx4", True, None, 2416, 9170, 3808), ("mx4", True, (8, 5), 1117, 1538, 448), ("mx4", False, None, 2384, 2472, 3648), ("mx4", True, None, 273, 6661, 10912),
         ("mx4", True, None, 42, 4110, 12896), ("mx4", False, (16, 4), 298, 1939, 3648), ("mx4", True, (16, 3), 2577, 338, 12576), ("16", True, (8, 5), 1117, 1538, 448),
         ("16", False, (16, 3), 2577, 1939, 3648), ("16", True, None, 273, 6661, 10912)]


def plan_of(kind, gated, units, n, N, K):
    """(rows, columns of a tile, slabs in LDS, K in pieces)"""
    from promoe_amd import _lib as L
    plan = (ctypes.c_int * 4)()
    assert L.lib.moe_mx4_plan(n, units, N, K, kind == "mx4", gated, ctypes.addressof(plan)) == 0
    return plan[0], plan[1], plan[2], plan[3] > 1


def key_of(case):
    kind, gated, by, n, N, K = case
    units, n = (0, n) if by is None else (min(by[0], n * by[1]), n * by[1])
    return (kind, gated, by is not None, *plan_of(kind, gated, units, n, N, K))


def test_every_kernel_of_the_plan_has_a_case():
    rng = random.Random(0)
    log = lambda low, high: int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    reached = set()
    for _ in range(100000):
        kind, gated, n, N, K = rng.choice(["mx4", "16"]), rng.random() < 0.5, log(1, 16384), log(1, 20000), 32 * log(1, 512)
        units = min(n, rng.choice([0, 0, 1, 2, 4, 8, 16, 60, 64, 256]))
        if units:
            n *= rng.randint(1, 4)
        reached.add((kind, gated, units > 0, *plan_of(kind, gated, units, n, N, K)))
    cases = [key_of(c) for c in CASES]
    assert len(set(cases)) == len(cases) == 72
    assert not reached - set(cases), sorted(reached - set(cases))


def test_plan_refuses_what_is_no_product():
    from promoe_amd import _lib as L
    plan = (ctypes.c_int * 4)()
    at = ctypes.addressof(plan)
    for args in ((0, 0, 8, 64, 0, 0, at), (4, -1, 8, 64, 0, 0, at), (4, 0, 0, 64, 0, 0, at), (4, 0, 8, 0, 0, 0, at), (4, 0, 8, 64, 0, 0, None)):
        assert L.lib.moe_mx4_plan(*args) == L.MOE_EINVAL and b"moe_mx4_plan" in L.lib.moe_last_error()


def beyond_fp16(q, gen, dev):
    """The same with scales among them whose codes are no fp16 values: in one row of each 16, all others as they were"""
    from promoe_amd import ops
    s = q.scales
    s[..., 5::16, -1] = 100
    s[..., 0, 0] = 101
    return ops.Mx4(q.codes, s)


def product(dev, case, dtype, far, seed):
    """far: some scales of W are outside of what fp16 weights can have"""
    from promoe_amd import ops
    kind, gated, by, n, N, K = case
    act, bias, out_dtype = ACTS[seed % 6], seed % 2 == 0, torch.float32 if seed % 3 == 2 else dtype
    print(f"case mx4_tile {case} {dtype} far={far} act={act} bias={bias} out={out_dtype} plan={key_of(case)[3:]}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(7 * n + N + K)
    E, k = (1, 1) if by is None else by
    of_tokens = by is not None and seed % 2 == 1
    M = n * k
    x = rows((n if of_tokens else M, K), 1.0, dtype, gen, dev, 8 * (seed % 2))
    xv = x.double()
    if kind == "mx4":
        x = ops.quantize_mx4(x)
        xv = values(x.codes, x.scales)
        x = spaced(x, seed % 2, dev)
    lead = () if by is None else (E,)
    mats = [matrix((*lead, N, K), gen, dev) for _ in range(2 if gated else 1)]
    if far:
        mats = [beyond_fp16(m, gen, dev) for m in mats]
    mats = [spaced(m, seed % 2, dev) for m in mats]
    bs = [rows((E, N), 0.5, dtype, gen, dev).contiguous().view(*lead, N) if bias else None for _ in mats]
    out = torch.full((M + 1, N + 3), 7.0, dtype=out_dtype, device=dev)
    y = out[:M, :N]
    if by is None:
        residual = rows((M, N), 1.0, dtype, gen, dev, seed % 3) if not gated and seed % 4 < 2 else None
        if gated:
            ops.linear_gated_mx4(x, *mats, *bs, act=act, out=y)
        else:
            ops.linear_mx4(x, mats[0], bs[0], act=act, residual=residual, out=y)
        torch.cuda.synchronize()
        want, err = expect(xv, [values(m.codes, m.scales) for m in mats], bs, act, residual)
        check(y, want, err)
        assert torch.all(out[M:] == 7.0) and torch.all(out[:, N:] == 7.0)
        return
    idx = torch.topk(torch.randn(n, E, device=dev, generator=gen) - torch.log1p(torch.arange(E, device=dev)), k, dim=1).indices.int().contiguous()
    by_expert(x, xv, mats, bs, idx, E, act, of_tokens, out)


def by_expert(x, xv, mats, bs, idx, E, act, of_tokens, out):
    from promoe_amd import ops
    T, k = idx.shape
    M, N = T * k, mats[0].shape[1]
    d = ops.dispatch(idx, E)
    (ops.experts_gated_mx4 if len(mats) == 2 else ops.experts_linear_mx4)(x, *mats, d, *bs, act=act, of_tokens=of_tokens, out=out[:M, :N])
    torch.cuda.synchronize()
    flat = idx.reshape(-1).cpu()
    at = 0
    for e in range(E):
        pairs = torch.nonzero(flat == e)[:, 0].to(idx.device)
        m = pairs.numel()
        if m:
            src = xv[pairs // k] if of_tokens else xv[at: at + m]
            check(out[at: at + m, :N], *expect(src, [values(q.codes[e], q.scales[e]) for q in mats], [b if b is None else b[e] for b in bs], act))
        at += m
    assert torch.all(out[at:] == 7.0) and torch.all(out[:, N:] == 7.0)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["bf16", "fp16", "fp16 far"])
@pytest.mark.parametrize("case", CASES + WIDER, ids=lambda c: "-".join(str(v).replace(" ", "") for v in c))
def test_every_kernel(cuda, case, how):
    if how == "fp16 far" and case[0] == "mx4":
        how = "fp16"                                      # (x in 4 bits meets any scale alike: another seed)
        seed = 3
    else:
        seed = 0
    product(cuda, case, torch.bfloat16 if how == "bf16" else torch.float16, how == "fp16 far", seed + (CASES + WIDER).index(case) + len(how))


COUNTS = [0, 1, 31, 32, 33, 63, 64, 65, 96, 97, 128, 129, 160, 161, 192, 193, 224, 225, 255, 256, 257, 289, 321, 512, 513, 700, 900, 1100, 1400, 0, 2, 1800]
COUNTED_N = 773


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True], ids=["linear", "gated"])
@pytest.mark.parametrize("of_tokens", [False, True], ids=["in order", "of tokens"])
@pytest.mark.parametrize("kind", ["mx4", "16"])
def test_experts_of_every_number_of_rows(cuda, kind, of_tokens, gated):
    """Tiles of 256 rows (x in 4 bits) that end after each of their blocks of 32, whole ones, experts of one row and of none."""
    from promoe_amd import ops
    E, T, N, K = len(COUNTS), sum(COUNTS), COUNTED_N, 288
    print(f"case mx4_counts {kind} gated={gated} of_tokens={of_tokens}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(11)
    idx = torch.repeat_interleave(torch.arange(E), torch.tensor(COUNTS))[torch.randperm(T, generator=torch.Generator().manual_seed(3))]
    x = rows((T, K), 1.0, torch.bfloat16, gen, cuda, 8)
    xv = x.double()
    if kind == "mx4":
        x = ops.quantize_mx4(x)
        xv = values(x.codes, x.scales)
    mats = [matrix((E, N, K), gen, cuda) for _ in range(2 if gated else 1)]
    bs = [rows((E, N), 0.5, torch.bfloat16, gen, cuda).contiguous() for _ in mats]
    out = torch.full((T + 1, N + 3), 7.0, dtype=torch.bfloat16, device=cuda)
    by_expert(x, xv, mats, bs, idx.int()[:, None].contiguous().to(cuda), E, "gelu_tanh", of_tokens, out)


def test_the_wide_kernel_takes_that_many_rows():
    for gated in (False, True):
        assert plan_of("mx4", gated, len(COUNTS), sum(COUNTS), COUNTED_N, 288)[:2] == (256, 256)


SPLIT = [(24, 2050, 10944), (60, 2050, 10944)]            # K in pieces: partial sums in a workspace of each call


def test_these_products_have_a_workspace():
    from promoe_amd import _lib as L
    for M, N, K in SPLIT:
        for x_mx4 in (0, 1):
            assert L.lib.moe_mx4_linear_workspace_bytes(M, N, K, x_mx4, 0) > 0 and L.lib.moe_mx4_linear_workspace_bytes(M, N, K, x_mx4, 1) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["mx4", "16"])
def test_partial_sums_of_two_streams_and_two_graphs(cuda, kind):
    """Products with K in pieces on two streams at once, and from two graphs replayed in turn and at once: the bits of one call by itself."""
    from promoe_amd import ops
    print(f"case mx4_pieces_at_once {kind}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(9)
    N, K = SPLIT[0][1:]
    w, w2 = matrix((N, K), gen, cuda), matrix((N, K), gen, cuda)
    q = ops.quantize_mx4 if kind == "mx4" else (lambda t: t)
    xs = [torch.randn(M, K, device=cuda, generator=gen).to(torch.bfloat16) for M, _, _ in SPLIT]
    block = lambda x: (ops.linear_mx4(q(x), w), ops.linear_gated_mx4(q(x), w, w2))
    want = [block(x) for x in xs]
    torch.cuda.synchronize()
    same = lambda a, b: all(torch.equal(p, r) for p, r in zip(a, b))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(block(xs[i]))
    torch.cuda.synchronize()
    assert all(same(g, want[i]) for i in range(2) for g in got[i])
    graphs, outs, ins = [], [], [x.clone() for x in xs]
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block(x))
        graphs.append(g)
    for i in range(4):
        for x, x0 in zip(ins, xs):
            x.copy_(x0 * (i + 1))
        torch.cuda.synchronize()
        if i % 2:
            for g in graphs:
                g.replay()
        else:
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for x, y in zip(ins, outs):
            assert same(y, block(x))
            torch.cuda.synchronize()
