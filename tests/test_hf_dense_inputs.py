"""Inputs and weights that the class's own forward of a dense layer takes and the fused products do not as they are."""
import types

import pytest
import torch
from torch import nn
from torch.nn import functional as F

from tests.test_hf_dense import Mlp, _found


def _inputs(H, dtype, dev):
    """(name, x): strided in ways that leave rows of H elements, or columns, apart."""
    gen = torch.Generator().manual_seed(3)

    def rand(*shape):
        return torch.randn(*shape, generator=gen).to(dtype).to(dev)
    yield "rows", rand(2, 5, H)
    yield "transposed", rand(1, H, 5).transpose(1, 2)
    yield "every second column", rand(2, 5, 2 * H)[..., ::2]
    yield "rows 8 further apart", rand(2, 5, H + 8)[..., :H]
    yield "rows an odd number apart", rand(2, 5, H + 3)[..., :H]
    yield "off a boundary", rand(2 * 5 * H + 1)[1:].view(2, 5, H)
    yield "one row for all", rand(1, 1, H).expand(2, 5, H)
    yield "a vector", rand(H)
    yield "one row, off a boundary", rand(H + 3)[3:]
    yield "none", rand(0, 5, H)


def _fuse(mlp):
    from promoe_amd import hf
    mlp.forward = types.MethodType(hf._fused_mlp_forward("silu", mlp.act_fn), mlp)
    return mlp


def test_what_reaches_the_products(monkeypatch):
    """On the CPU, with stand-ins for the two products that refuse what they refuse."""
    from promoe_amd import hf

    def check(x, *w):
        assert x.dim() == 2 and x.dtype == w[0].dtype and x.data_ptr() % 16 == 0
        assert x.stride(1) == 1 and (x.shape[0] < 2 or (x.stride(0) % 8 == 0 and x.shape[1] <= x.stride(0) < 1 << 21))

    def gated(x, wg, wu, bg, bu, act):
        check(x, wg)
        return F.silu(F.linear(x, wg, bg)) * F.linear(x, wu, bu)

    def linear(x, w, b):
        check(x, w)
        return F.linear(x, w, b)
    monkeypatch.setattr(hf.ops, "linear_gated", gated)
    monkeypatch.setattr(hf.ops, "linear", linear)
    mlp = _fuse(Mlp())
    for name, x in _inputs(32, torch.float32, "cpu"):
        y, ref = mlp(x), Mlp.forward(mlp, x)
        assert y.shape == ref.shape and torch.allclose(y, ref, atol=1e-6), name
    with torch.autocast("cpu", dtype=torch.bfloat16):                # (the class's own products, whatever the types)
        mlp = _fuse(Mlp().to(torch.bfloat16))
        x = torch.randn(2, 5, 32)
        assert torch.equal(mlp(x), Mlp.forward(mlp, x))


def test_weights_off_a_boundary_or_of_other_strides_are_left(monkeypatch):
    off, turned = Mlp(), Mlp()
    off.up_proj.weight = nn.Parameter(torch.zeros(32 * 64 + 1)[1:].view(64, 32))
    turned.down_proj.weight = nn.Parameter(torch.zeros(64, 32).t())
    assert _found(monkeypatch, off=off, turned=turned, fine=Mlp()) == {"fine": "silu"}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fused_layer_on_such_inputs(cuda, dtype):
    """Against the class's own forward in 64 bits: the intermediate rounded once, then the result (eps / 2 each; sums in fp32)."""
    torch.manual_seed(5)
    mlp = _fuse(Mlp(H=64, I=120, act=nn.SiLU()).to(dtype).to(cuda))
    eps = torch.finfo(dtype).eps / 2
    wg, wu, wd = (p.weight.detach().double().cpu() for p in (mlp.gate_proj, mlp.up_proj, mlp.down_proj))
    for name, x in _inputs(64, dtype, cuda):
        print(f"case fused_inputs {dtype} {name}", flush=True)
        y = mlp(x)
        assert y.shape == x.shape and y.dtype == dtype
        xd = x.double().cpu()
        h = F.silu(xd @ wg.t()) * (xd @ wu.t())
        ref = h @ wd.t()
        tol = 1.01 * eps * ((h.abs() + torch.finfo(dtype).tiny) @ wd.abs().t() + ref.abs()) + 1e-6
        assert ((y.double().cpu() - ref).abs() <= tol).all(), name
