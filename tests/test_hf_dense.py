"""Which layers of a model the fused products take, which routers become a rule, and what set_layer refuses (no GPU needed)."""
import types

import pytest
import torch
from torch import nn


class Mlp(nn.Module):
    def __init__(self, H=32, I=64, act=nn.SiLU(), linear=nn.Linear, **more):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj = linear(H, I, bias=False), linear(H, I, bias=False), linear(I, H, bias=False)
        self.act_fn = act
        for n, m in more.items():
            setattr(self, n, m)

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class PackedLinear(nn.Linear):
    """A product of its own, as quantised layers and layers with adapters are."""


class Relu2(nn.Module):
    def forward(self, x):
        return x.relu() ** 2


def _found(monkeypatch, **mods):
    from promoe_amd import hf
    monkeypatch.setattr(hf, "find_moe_blocks", lambda model: [])
    return {n: a for n, _, a in hf.find_dense_mlps(nn.ModuleDict(mods))}


def test_activations_are_told_by_their_values(monkeypatch):
    acts = dict(silu=nn.SiLU(), gelu=nn.GELU(), gelu_tanh=nn.GELU(approximate="tanh"), relu=nn.ReLU(), relu2=Relu2())
    assert _found(monkeypatch, **{n: Mlp(act=a) for n, a in acts.items()}) == {n: n for n in acts}
    assert _found(monkeypatch, a=Mlp(act=nn.Tanh()), b=Mlp(act=nn.PReLU()), c=Mlp(act=None), d=Mlp(act=nn.LeakyReLU())) == {}


def test_layers_that_are_more_than_three_plain_products_are_left(monkeypatch):
    hooked, replaced, inner = Mlp(), Mlp(), Mlp()
    hooked.up_proj.register_forward_hook(lambda m, a, y: 2 * y)
    replaced.forward = types.MethodType(lambda self, x: x, replaced)
    inner.down_proj.forward = types.MethodType(lambda self, x: x, inner.down_proj)
    assert _found(monkeypatch, packed=Mlp(linear=PackedLinear), norm=Mlp(norm=nn.LayerNorm(64)), hooked=hooked, replaced=replaced, inner=inner,
                  odd=Mlp(I=60), odd_h=Mlp(H=36), fine=Mlp()) == {"fine": "silu"}


def test_routers_that_no_rule_describes_are_refused():
    from promoe_amd import hf
    bias = dict(e_score_correction_bias=torch.zeros(16), n_group=4, topk_group=2, norm_topk_prob=True, routed_scaling_factor=2.5)
    rule, b = hf._route_rule(types.SimpleNamespace(gate=types.SimpleNamespace(**bias)))
    assert rule.n_group == 4 and rule.renorm == 1 and b is bias["e_score_correction_bias"]
    for more in (dict(bias, scoring_func="softmax"), dict(bias, score_function="softmax"),
                 dict(topk_method="group_limited_greedy", num_group=4, topk_group=2, routed_scaling_factor=1.0, norm_topk_prob=True)):
        with pytest.raises(NotImplementedError):
            hf._route_rule(types.SimpleNamespace(gate=types.SimpleNamespace(**more)))


def test_set_layer_refuses_a_bias_without_a_rule_and_a_bad_rule_before_the_layer_is_described():
    from promoe_amd import _lib as L
    from promoe_amd import engine, ops
    pm = engine.PrefetchMngr.__new__(engine.PrefetchMngr)        # (neither call gets as far as an engine)
    pm._keep, pm._h = [], None
    gate = torch.zeros(16, 256, dtype=torch.bfloat16)
    rule = ops.RouteRule("sigmoid", 4, 2, "top2")
    for kw in (dict(select_bias=torch.zeros(16)), dict(rule=rule, select_bias=torch.zeros(15)),
               dict(rule=rule, select_bias=torch.zeros(16, dtype=torch.bfloat16)), dict(rule=ops.RouteRule("sigmoid", 3, 2)),
               dict(rule=ops.RouteRule("softmax", 4, 5)), dict(rule=ops.RouteRule("softmax", 16, 2))):
        with pytest.raises(L.MoeError):
            pm.set_layer(0, 256, 128, 0, 4, 0, gate, **kw)
        assert not pm._keep
