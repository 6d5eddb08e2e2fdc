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


def _mlp(forward, **attrs):
    m = type("M", (Mlp,), {"forward": forward})()
    for n, v in attrs.items():
        setattr(m, n, v)
    return m


def test_a_forward_of_another_form_is_left(monkeypatch):
    """Factors, clips and selections that are plain attributes of the module or constants of its class."""
    others = dict(
        factor=_mlp(lambda s, x: s.down_proj(s.act_fn(s.gate_proj(x) * s.m) * s.up_proj(x)), m=1.01),
        out_factor=_mlp(lambda s, x: s.down_proj(s.act_fn(s.gate_proj(x)) * s.up_proj(x)) * s.m, m=nn.Parameter(torch.tensor(0.5))),
        clip_gate=_mlp(lambda s, x: s.down_proj(s.act_fn(s.gate_proj(x).clamp(max=s.limit)) * s.up_proj(x)), limit=10.0),
        clip_up=_mlp(lambda s, x: s.down_proj(s.act_fn(s.gate_proj(x)) * s.up_proj(x).clamp(-7, 7))),
        up_plus_one=_mlp(lambda s, x: s.down_proj(s.act_fn(s.gate_proj(x)) * (s.up_proj(x) + 1))),
        swapped=_mlp(lambda s, x: s.down_proj(s.act_fn(s.up_proj(x)) * s.gate_proj(x))),
        added=_mlp(lambda s, x: x + s.down_proj(s.act_fn(s.gate_proj(x)) * s.up_proj(x))),
        sparse=_mlp(lambda s, x: s.down_proj(s.act_fn(F.relu(s.gate_proj(x) - s.gate_proj(x).std(-1, keepdim=True))) * s.up_proj(x))),
        last_column=_mlp(lambda s, x: s.down_proj(torch.cat([(h := s.act_fn(s.gate_proj(x)) * s.up_proj(x))[..., :-1], 0 * h[..., -1:]], -1))),
        more_arguments=_mlp(lambda s, x, y: s.down_proj(s.act_fn(s.gate_proj(x)) * s.up_proj(x)) + y),
        pair=_mlp(lambda s, x: (s.down_proj(s.act_fn(s.gate_proj(x)) * s.up_proj(x)), None)),
        by_weight=_mlp(lambda s, x: s.down_proj(s.act_fn(F.linear(x, s.gate_proj.weight)) * s.up_proj(x))),
    )
    assert _found(monkeypatch, **others) == {}
    same = dict(up_first=_mlp(lambda s, x: s.down_proj(s.up_proj(x) * s.act_fn(s.gate_proj(x)))),
                typed=_mlp(lambda s, x: s.down_proj(s.act_fn(s.gate_proj(x.to(s.gate_proj.weight.dtype))) * s.up_proj(x))),
                rows=_mlp(lambda s, x: s.down_proj(s.act_fn(s.gate_proj(x.reshape(-1, x.shape[-1]))) * s.up_proj(x.reshape(-1, x.shape[-1]))).view(x.shape)),
                narrow=Mlp(H=64, I=24), bf16=Mlp().to(torch.bfloat16), short=Mlp(I=40))
    assert _found(monkeypatch, **same) == {n: "silu" for n in same}
    # (nothing of the module has changed)
    m = Mlp()
    before = {n: t.clone() for n, t in m.state_dict().items()}
    _found(monkeypatch, m=m)
    assert type(m.gate_proj) is nn.Linear and all(torch.equal(m.state_dict()[n], t) for n, t in before.items())


def test_a_hook_on_the_activation_is_left(monkeypatch):
    hooked, early, replaced = (Mlp(act=nn.SiLU()) for _ in range(3))  # (an activation of its own each)
    hooked.act_fn.register_forward_hook(lambda m, a, y: 2 * y)
    seen = []
    early.act_fn.register_forward_pre_hook(lambda m, a: seen.append(a[0].shape))
    replaced.act_fn.forward = lambda x: F.silu(x)
    assert _found(monkeypatch, hooked=hooked, early=early, replaced=replaced, fine=Mlp(), function=Mlp(act=F.silu)) == {"fine": "silu", "function": "silu"}


def test_what_is_changed_after_the_injection_has_its_effect(monkeypatch):
    """Hooks, replaced parts and forwards put on a fused layer later: the class's own forward runs, and the fused products again when
    they are gone."""
    import types

    from promoe_amd import hf
    calls = []

    def gated(x, wg, wu, bg, bu, act):
        calls.append("gated")
        return F.silu(F.linear(x, wg, bg)) * F.linear(x, wu, bu)
    monkeypatch.setattr(hf.ops, "linear_gated", gated)
    monkeypatch.setattr(hf.ops, "linear", F.linear)
    torch.manual_seed(2)
    mlp, x = Mlp(act=nn.SiLU()), torch.randn(2, 5, 32)
    plain = mlp(x).detach()
    mlp.forward = types.MethodType(hf._fused_mlp_forward("silu", mlp.act_fn), mlp)

    def fused():
        calls.clear()
        y = mlp(x)
        return y.detach(), bool(calls)

    def unchanged():
        y, f = fused()
        return f and torch.allclose(y, plain, atol=1e-6)
    assert unchanged()
    for part in ("gate_proj", "up_proj", "down_proj", "act_fn"):
        handle = getattr(mlp, part).register_forward_hook(lambda m, a, y: 2 * y)
        y, f = fused()
        assert not f and torch.allclose(y, 2 * plain, atol=1e-5) == (part != "gate_proj")
        handle.remove()
        assert unchanged()
    handle = mlp.up_proj.register_forward_pre_hook(lambda m, a: (a[0] * 2,))
    y, f = fused()
    assert not f and torch.allclose(y, 2 * plain, atol=1e-5)
    handle.remove()

    class Adapter(nn.Linear):
        def forward(self, v):
            return 3 * super().forward(v)
    own = mlp.down_proj
    mlp.down_proj = Adapter(64, 32, bias=False)
    mlp.down_proj.weight = own.weight
    y, f = fused()
    assert not f and torch.allclose(y, 3 * plain, atol=1e-5)
    mlp.down_proj = own
    act = mlp.act_fn
    mlp.act_fn = nn.ReLU()
    y, f = fused()
    assert not f and torch.allclose(y, Mlp.forward(mlp, x), atol=1e-6)
    mlp.act_fn = act
    assert unchanged()
    # (other weights in the same parts are no other form)
    mlp.down_proj.weight = nn.Parameter(2 * own.weight.detach())
    y, f = fused()
    assert f and torch.allclose(y, 2 * plain, atol=1e-5)
