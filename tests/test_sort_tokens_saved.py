"""The backward pass of unsort_tokens reads the saved rows as a saved-tensor hook returns them.

Without a GPU: the library is replaced by a recorder, so that nothing is read, and what the kernel would be told is compared with the
tensors that the hook returned."""
import pytest
import torch

T, H, K = 3, 16, 2


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


def backward(monkeypatch, x, w, pack, unpack):
    """(result of the backward pass, arguments of the gradient's launch)"""
    from promoe_amd import ops
    lib = Recorder()
    monkeypatch.setattr(ops, "lib", lib)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)
    d = ops.Dispatch(T, K, 4, 4, "cpu")
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y = ops._UnsortTokens.apply(x, w, d, x.stride(0))
    grads = torch.autograd.grad(y, [x, w], torch.ones(T, H, dtype=x.dtype))
    (args,) = [a for name, a in lib.calls if name == "moe_unsort_rows_grad"]
    return grads, args


def leaves(ld):
    x = torch.randn(T * K, ld).to(torch.bfloat16)[:, :H].requires_grad_(True)
    return x, torch.rand(T, K, requires_grad=True)


@pytest.mark.parametrize("laid_out", [lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format),
                                      lambda t: torch.nn.functional.pad(t, (0, 40))[:, : t.shape[1]], lambda t: t.t().contiguous().t(),
                                      lambda t: t[:1].clone().expand(t.shape[0], -1)],
                         ids=["as saved", "contiguous", "further apart", "columns whole", "one row"])
@pytest.mark.parametrize("ld", [H, 24])
def test_rows_as_the_hook_returns_them(monkeypatch, ld, laid_out):
    given = []

    def unpack(t):
        t = laid_out(t.detach())
        given.append(t)
        return t

    x, w = leaves(ld)
    _, args = backward(monkeypatch, x, w, lambda t: t, unpack)
    rows, weights = given[-2:]
    _, _, x_ptr, ldx, _, w_ptr = args[:6]
    if rows.stride(1) == 1 and rows.stride(0) >= H:
        assert x_ptr == rows.data_ptr() and ldx == rows.stride(0)
    else:                                                     # (a copy of its own)
        assert x_ptr != rows.data_ptr() and ldx == H
    assert (w_ptr == weights.data_ptr()) == weights.is_contiguous()


@pytest.mark.parametrize("spoil", [lambda t: t.double() if t.dtype == torch.bfloat16 else t, lambda t: t.half() if t.dtype == torch.float32 else t,
                                   lambda t: t[:-1], lambda t: t[:, :-1], lambda t: t.flatten()],
                         ids=["rows of another type", "weights of another type", "fewer rows", "fewer columns", "no matrix"])
def test_other_types_and_sizes_are_refused(monkeypatch, spoil):
    from promoe_amd import _lib as L
    x, w = leaves(24)
    with pytest.raises(L.MoeError, match="unsort_tokens"):
        backward(monkeypatch, x, w, lambda t: t, lambda t: spoil(t.detach()))


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [0, 8])
def test_gradients_of_rows_kept_elsewhere(cuda, gap):
    """Rows kept in host memory between forward and backward, and rows that a hook lays out anew: the same bits as of rows that lie so
    without a hook (the order in which a weight's gradient is added up goes by the rows' alignment)."""
    from promoe_amd import ops
    T, H, k, E = 65, 72, 3, 8
    gen = torch.Generator(device=cuda).manual_seed(gap)
    d = ops.dispatch(torch.topk(torch.randn(T, E, device=cuda, generator=gen), k, dim=1).indices.int().contiguous(), E)
    x = torch.randn(T * k, H + gap, device=cuda, generator=gen).to(torch.bfloat16)[:, :H].requires_grad_(True)
    w = torch.rand(T, k, device=cuda, generator=gen).requires_grad_(True)
    g = torch.randn(T, H, device=cuda, generator=gen).to(torch.bfloat16)
    hooks = torch.autograd.graph.saved_tensors_hooks
    whole, apart = lambda t: t.detach().contiguous(), lambda t: torch.nn.functional.pad(t.detach(), (0, 9))[:, : t.shape[1]]
    for name, kept, laid_out in (("on the CPU", torch.autograd.graph.save_on_cpu(), whole),
                                 ("to the CPU and back", hooks(lambda t: t.detach().cpu(), lambda t: t.to(cuda)), whole),
                                 ("apart", hooks(lambda t: t, lambda t: apart(t) if t.dtype == torch.bfloat16 else t), apart)):
        print(f"case unsort_saved gap={gap} {name}", flush=True)
        with kept:
            y = ops.unsort_tokens(x, d, w)
        dx, dw = torch.autograd.grad(y, [x, w], g)
        torch.cuda.synchronize()
        xl, wl = laid_out(x).requires_grad_(True), w.detach().clone().requires_grad_(True)
        want = torch.autograd.grad(ops.unsort_tokens(xl, d, wl), [xl, wl], g)
        assert torch.equal(dx, want[0]), "rows"
        assert torch.equal(dw, want[1]), "weights"
