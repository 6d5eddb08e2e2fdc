"""Dense gated layers that look like one of the fused form and are not: left with the module's own operations (no GPU needed)."""
import pytest
import torch
from torch import nn
from torch.nn import functional as F

from tests.test_hf_dense import Mlp, _found


class Of(nn.Module):
    def __init__(self, fn):
        super().__init__()
        self.fn = fn

    def forward(self, x):
        return self.fn(x)


def test_clipped_activations_are_others(monkeypatch):
    clipped = dict(relu6=nn.ReLU6(), gelu_10=Of(lambda x: F.gelu(x).clamp(-10, 10)), silu_100=Of(lambda x: F.silu(x.clamp(max=100.0))),
                   silu_low=Of(lambda x: F.silu(x.clamp(min=-5.0))), relu_1000=Of(lambda x: x.relu().clamp(max=1000.0)),
                   late=Of(lambda x: F.silu(x) + (x.abs() > 7).to(x.dtype) * 0.01))
    assert _found(monkeypatch, **{n: Mlp(act=a) for n, a in clipped.items()}) == {}
    # the same functions in other words are the same
    same = dict(silu=Of(lambda x: x * torch.sigmoid(x)), gelu=Of(lambda x: x * 0.5 * (1 + torch.erf(x / 2 ** 0.5))), relu=Of(lambda x: x.clamp(min=0)),
                gelu_tanh=Of(lambda x: 0.5 * x * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)))),
                relu2=Of(lambda x: F.relu(x).square()))
    assert _found(monkeypatch, **{n: Mlp(act=a) for n, a in same.items()}) == {n: n for n in same}


def test_activations_of_transformers(monkeypatch):
    acts = pytest.importorskip("transformers.activations").ACT2FN
    names = [n for n in ("relu6", "gelu_10", "quick_gelu", "tanh", "sigmoid", "leaky_relu", "mish") if n in acts]
    assert _found(monkeypatch, **{n: Mlp(act=acts[n]) for n in names}) == {}
    known = {"silu": "silu", "swish": "silu", "gelu": "gelu", "gelu_new": "gelu_tanh", "gelu_pytorch_tanh": "gelu_tanh", "relu": "relu", "relu2": "relu2"}
    known = {n: a for n, a in known.items() if n in acts}
    assert _found(monkeypatch, **{n: Mlp(act=acts[n]) for n in known}) == known
