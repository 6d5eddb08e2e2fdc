"""Tokens sorted by expert and back on the GPU, and the gradients, against the formulas in 64 bits and against differences.

Tolerances.  Sorting copies: equal.  A sum of k products of fp32 weights and values rounds at most k times by 2^-24 of the sum of
magnitudes (a fused product and addition rounds once), then once to the result's type (half a step).  A weight's gradient sums H products
in fp32: 256 lanes of at most ceil(H / 256) steps and the joins (at most 10 more), e = (H / 256 + 12) 2^-24 sum |dy x|, twice that counted."""
import pytest
import torch

from tests.test_linear_gpu import check, rows

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [(1, 1, 1, 4), (1, 2048, 6, 64), (2, 7, 2, 8), (3, 8, 3, 8), (33, 3584, 8, 64), (37, 100, 5, 60), (64, 4096, 1, 8), (100, 24, 7, 256),
          (129, 1030, 9, 32), (200, 72, 20, 64), (500, 2048, 4, 60), (1000, 264, 2, 8), (1, 30000, 8, 8)]


def routing(T, k, E, gen, dev, left):
    from promoe_amd import ops
    idx = torch.topk(torch.randn(T, E, device=dev, generator=gen), k, dim=1).indices.int()
    if left:
        idx[torch.rand(T, k, device=dev, generator=gen) < left] = -1
    flat = idx.reshape(-1).cpu()
    pairs = torch.cat([torch.nonzero(flat == e)[:, 0] for e in range(E)]).to(dev)      # the pair of each row
    return ops.dispatch(idx.contiguous(), E), pairs


@pytest.mark.parametrize("left", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("T,H,k,E", SHAPES)
def test_there_and_back_with_gradients(cuda, T, H, k, E, left):
    from promoe_amd import ops
    i = SHAPES.index((T, H, k, E))
    dtype = TYPES[i % 3]
    for gap in (0, 3, 8):
        print(f"case sort T={T} H={H} k={k} E={E} {dtype} left={left} gap={gap}", flush=True)
        gen = torch.Generator(device=cuda).manual_seed(T + H + k)
        d, pairs = routing(T, k, E, gen, cuda, left)
        P, n, tok = T * k, pairs.numel(), pairs // k
        # there
        x = rows((T, H), 1.0, dtype, gen, cuda, gap).requires_grad_(True)
        y = ops.sort_tokens(x, d)
        want = torch.zeros(P, H, dtype=dtype, device=cuda)
        want[:n] = x.detach()[tok]
        assert torch.equal(y.detach(), want)
        assert torch.equal(ops.sort_tokens(x.detach(), d), want)
        g = rows((P, H), 1.0, dtype, gen, cuda, gap)
        (dx,) = torch.autograd.grad(y, [x], g)
        z = lambda: torch.zeros(T, H, dtype=torch.float64, device=cuda)
        check(dx, z().index_add_(0, tok, g.double()[:n]), k * 2.0 ** -24 * z().index_add_(0, tok, g.double().abs()[:n]))
        # back, what lies behind the last row being NaN
        r = rows((P, H), 1.0, dtype, gen, cuda, gap)
        r[n:] = float("nan")
        r.requires_grad_(True)
        w = torch.rand(T, k, device=cuda, generator=gen).requires_grad_(True)
        y = ops.unsort_tokens(r, d, w)
        rv, wv = r.detach().double()[:n], w.detach().double().reshape(-1)[pairs, None]
        check(y.detach(), z().index_add_(0, tok, rv * wv), k * 2.0 ** -24 * z().index_add_(0, tok, (rv * wv).abs()))
        g = rows((T, H), 1.0, dtype, gen, cuda, gap)
        dr, dw = torch.autograd.grad(y, [r, w], g)
        want = torch.zeros(P, H, dtype=torch.float64, device=cuda)
        want[:n] = g.double()[tok] * wv
        check(dr, want, 2.0 ** -24 * want.abs())
        ref, mag = (torch.zeros(P, dtype=torch.float64, device=cuda) for _ in range(2))
        ref[pairs] = (g.double()[tok] * rv).sum(1)
        mag[pairs] = (g.double()[tok] * rv).abs().sum(1)
        assert dw.shape == (T, k) and ((dw.double() - ref.view(T, k)).abs() <= 2 * (H / 256 + 12) * 2.0 ** -24 * mag.view(T, k)).all()
        # one gradient without the other; sums without weights
        y = ops.unsort_tokens(r.detach(), d, w)
        assert torch.equal(torch.autograd.grad(y, [w], g)[0], dw)
        y = ops.unsort_tokens(r, d, w.detach())
        assert torch.equal(torch.autograd.grad(y, [r], g)[0], dr)
        y = ops.unsort_tokens(r, d)
        check(y.detach(), z().index_add_(0, tok, rv), k * 2.0 ** -24 * z().index_add_(0, tok, rv.abs()))
        (dr,) = torch.autograd.grad(y, [r], g)
        want = torch.zeros(P, H, dtype=dtype, device=cuda)
        want[:n] = g[tok]
        assert torch.equal(dr, want)


def test_gradients_against_differences(cuda):
    """A scalar of there, a product per row, and back, along random directions: (f(a + h) - f(a - h)) / 2h in fp32.  f is of degree two in
    (x, w), so the difference has no error but rounding: 2^-24 of about sqrt(4 * 240) terms of size 1 over h = 2^-4, below 1e-3 of f's scale 31."""
    from promoe_amd import ops
    print("case sort_differences", flush=True)
    T, H, k, E = 20, 12, 3, 8
    gen = torch.Generator(device=cuda).manual_seed(4)
    d, _ = routing(T, k, E, gen, cuda, 0.2)
    x = torch.randn(T, H, device=cuda, generator=gen)
    w = torch.rand(T, k, device=cuda, generator=gen)
    c, g = torch.randn(T * k, H, device=cuda, generator=gen), torch.randn(T, H, device=cuda, generator=gen)

    def f(x, w):
        return (ops.unsort_tokens(ops.sort_tokens(x, d) * c, d, w) * g).sum()

    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(f(xl, wl), [xl, wl])
    h = 2.0 ** -4
    for _ in range(4):
        vx, vw = torch.randn(T, H, device=cuda, generator=gen), torch.randn(T, k, device=cuda, generator=gen)
        slope_ = (gx.double() * vx).sum() + (gw.double() * vw).sum()
        diff = (f(x + h * vx, w + h * vw).double() - f(x - h * vx, w - h * vw).double()) / (2 * h)
        assert abs(float(diff - slope_)) <= 1e-3 * 31, (float(diff), float(slope_))


def test_a_strange_gradient_streams_graphs_and_refusals(cuda):
    from promoe_amd import _lib as L
    from promoe_amd import ops
    print("case sort_more", flush=True)
    T, H, k, E = 50, 64, 4, 16
    gen = torch.Generator(device=cuda).manual_seed(4)
    d, _ = routing(T, k, E, gen, cuda, 0.0)
    x = torch.randn(T, H, device=cuda, generator=gen).to(torch.bfloat16)
    w = torch.rand(T, k, device=cuda, generator=gen)
    # an expanded gradient, a transposed one
    xl = x.clone().requires_grad_(True)
    ops.sort_tokens(xl, d).sum().backward()
    assert torch.equal(xl.grad, torch.full_like(x, k))
    r = torch.randn(T * k, H, device=cuda, generator=gen).to(torch.bfloat16)
    rl, wl = r.clone().requires_grad_(True), w.clone().requires_grad_(True)
    turned = torch.randn(H, T, device=cuda, generator=gen).to(torch.bfloat16).t()
    a = torch.autograd.grad(ops.unsort_tokens(rl, d, wl), [rl, wl], turned)
    b = torch.autograd.grad(ops.unsort_tokens(rl, d, wl), [rl, wl], turned.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # no second gradient
    with pytest.raises(L.MoeError, match="second"):
        torch.autograd.grad(ops.sort_tokens(xl, d), [xl], torch.ones_like(r), create_graph=True)
    with pytest.raises(L.MoeError, match="second"):
        torch.autograd.grad(ops.unsort_tokens(rl, d, wl), [rl], torch.ones_like(x), create_graph=True)
    # the same bits every time, on another stream and from a graph
    want = ops.unsort_tokens(ops.sort_tokens(x, d), d, w)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        assert torch.equal(ops.unsort_tokens(ops.sort_tokens(x, d), d, w), want)
    torch.cuda.synchronize()
    xg = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.unsort_tokens(ops.sort_tokens(xg, d), d, w)
    for i in range(4):
        xg.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.unsort_tokens(ops.sort_tokens(xg, d), d, w))
    assert ops.sort_tokens(torch.empty(T, 0, device=cuda), d).shape == (T * k, 0)
    for call in (lambda: ops.sort_tokens(x[:-1], d), lambda: ops.sort_tokens(x.double(), d), lambda: ops.sort_tokens(x.cpu(), d),
                 lambda: ops.sort_tokens(x[None], d), lambda: ops.unsort_tokens(x, d), lambda: ops.unsort_tokens(r, d, w[:, :2]),
                 lambda: ops.unsort_tokens(r, d, w.half()), lambda: ops.unsort_tokens(r, d, w.t().contiguous().t()),
                 lambda: ops.unsort_tokens(r.t().contiguous().t(), d, w), lambda: ops.unsort_tokens(r, d, w.cpu())):
        with pytest.raises(L.MoeError):
            call()


def test_rows_far_apart(cuda):
    """Rows 6 MiB apart: offsets pass 2^32 bytes."""
    from promoe_amd import ops
    print("case sort_far", flush=True)
    T, H, k, E, ld = 400, 40, 2, 8, 3 << 20
    gen = torch.Generator(device=cuda).manual_seed(4)
    d, _ = routing(T, k, E, gen, cuda, 0.0)

    def far(t):
        v = torch.empty((t.shape[0] - 1) * ld + t.shape[1], dtype=t.dtype, device=cuda).as_strided(t.shape, (ld, 1))
        v.copy_(t)
        return v

    x, r = torch.randn(T, H, device=cuda, generator=gen).to(torch.bfloat16), torch.randn(T * k, H, device=cuda, generator=gen).to(torch.bfloat16)
    w = torch.rand(T, k, device=cuda, generator=gen)
    assert torch.equal(ops.sort_tokens(far(x), d), ops.sort_tokens(x, d))
    fr, wl, rl = far(r).requires_grad_(True), w.clone().requires_grad_(True), r.clone().requires_grad_(True)
    a, b = ops.unsort_tokens(fr, d, wl), ops.unsort_tokens(rl, d, wl)
    assert torch.equal(a, b)
    ga, gb = torch.autograd.grad(a, [fr, wl], far(x)), torch.autograd.grad(b, [rl, wl], x)
    assert all(torch.equal(p, q) for p, q in zip(ga, gb))


@pytest.mark.parametrize("T,k,E", [(5, 2, 4), (300, 4, 60), (700, 3, 64), (3000, 8, 256), (1500, 2, 700)])
def test_choices_of_no_expert_have_no_place(cuda, T, k, E):
    """From every dispatch that takes indices: places of the others as without them, -1 for theirs."""
    from promoe_amd import ops
    print(f"case no_expert T={T} k={k} E={E}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(T)
    for single in (False, True):
        idx = torch.randint(-2, E + 2, (T, k), device=cuda, generator=gen, dtype=torch.int32)
        d = ops.dispatch(idx, E, single_workgroup=single)
        torch.cuda.synchronize()
        d.check()
        flat = idx.reshape(-1).long()
        ok = (flat >= 0) & (flat < E)
        order = torch.sort(torch.where(ok, flat, E), stable=True).indices
        n = int(ok.sum())
        pos = torch.full((T * k,), -1, dtype=torch.int32, device=cuda)
        pos[order[:n]] = torch.arange(n, dtype=torch.int32, device=cuda)
        assert int(d.offsets[E]) == n and torch.equal(d.pos_of_pair, pos) and torch.equal(d.sorted_pair[:n].long(), order[:n])


def test_weights_of_rows_without_columns(cuda):
    """Rows of no columns: nothing but the weights' gradient, which is zero."""
    from promoe_amd import ops
    print("case unsort_no_columns", flush=True)
    T, k, E = 9, 3, 4
    gen = torch.Generator(device=cuda).manual_seed(6)
    d, _ = routing(T, k, E, gen, cuda, 0.0)
    r = torch.empty(T * k, 0, device=cuda, requires_grad=True)
    w = torch.ones(T, k, device=cuda, requires_grad=True)
    y = ops.unsort_tokens(r, d, w)
    dr, dw = torch.autograd.grad(y, [r, w], torch.empty_like(y))
    assert y.shape == (T, 0) and dr.shape == r.shape and dw.shape == w.shape and not dw.any()


def test_there_and_back_captured_with_gradients(cuda):
    """Forward and backward in one graph, replayed with new values between eager runs on other leaves: the same bits."""
    from promoe_amd import ops
    print("case moves_captured_backward", flush=True)
    T, H, k, E = 65, 72, 3, 8
    gen = torch.Generator(device=cuda).manual_seed(7)
    d, _ = routing(T, k, E, gen, cuda, 0.2)
    x0, g0 = (rows((T, H), 1.0, torch.bfloat16, gen, cuda) for _ in range(2))
    w0 = torch.rand(T, k, device=cuda, generator=gen)

    def step(x, w, g):
        y = ops.unsort_tokens(ops.sort_tokens(x, d), d, w)
        return (y.detach(), *torch.autograd.grad(y, [x, w], g))

    def eager(x, w, g):
        return step(x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_(), g.clone())

    x, w, g = x0.clone().requires_grad_(), w0.clone().requires_grad_(), g0.clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(2):
            step(x, w, g)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, w, g)
    for i in range(4):
        with torch.no_grad():
            x.copy_(x0 * (i + 1))
            w.copy_(w0 + i)
            g.copy_(g0 * (2 - i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager(x, w, g)))
