"""Stock sparse blocks: what hf.py reads out of their routers against the block's own forward on the CPU, and which are refused
(no GPU needed)."""
import pytest
import torch
from torch import nn

transformers = pytest.importorskip("transformers")

SIZES = dict(vocab_size=64, hidden_size=64, intermediate_size=64, moe_intermediate_size=64, num_hidden_layers=2, num_attention_heads=4,
             num_key_value_heads=4, first_k_dense_replace=0, n_group=4, topk_group=2, head_dim=16, max_position_embeddings=64, kv_lora_rank=16,
             q_lora_rank=16, qk_rope_head_dim=16, qk_nope_head_dim=16, v_head_dim=16, moe_layer_start_index=0, pad_token_id=0,
             n_routed_experts=16, num_experts=16, num_local_experts=16, moe_num_experts=16, num_experts_per_tok=4, moe_k=4)


def _blocks(name, **more):
    """The sparse blocks of a small model of a transformers family, with weights that tell experts apart."""
    from promoe_amd import hf
    make, config = getattr(transformers, name + "ForCausalLM", None), getattr(transformers, name + "Config", None)
    if make is None or config is None:
        pytest.skip("this transformers has no " + name)
    known = config()
    cfg = config(**{k: v for k, v in dict(SIZES, **more).items() if hasattr(known, k)})
    torch.manual_seed(0)
    model = make(cfg).eval()
    blocks = [b for _, b in hf.find_moe_blocks(model)]
    assert blocks
    with torch.no_grad():
        for b in blocks:
            for n, t in b.state_dict(keep_vars=True).items():
                if n.endswith("correction_bias"):
                    t.copy_(torch.randn_like(t) * 0.3)
                elif t.is_floating_point():
                    t.copy_(torch.randn_like(t) * (0.3 if n == "gate.weight" else 0.1))
    return model, blocks


@pytest.mark.parametrize("name", ["MiniMaxM2", "HYV3", "Ernie4_5_Moe"])
def test_a_selection_bias_that_is_not_on_the_gate_is_refused(name):
    from promoe_amd import hf
    model, blocks = _blocks(name)
    for b in blocks:
        with pytest.raises(NotImplementedError, match="e_score_correction_bias"):
            hf._route_rule(b)


def test_a_bias_on_any_module_of_a_block_is_refused():
    from promoe_amd import hf

    class Block(nn.Module):
        def __init__(self, where):
            super().__init__()
            self.gate, self.experts = nn.Linear(8, 4, bias=False), nn.Module()
            self.gate.top_k = 2
            self.gate.inner = nn.Module()
            at = {"block": self, "experts": self.experts, "inner": self.gate.inner, None: nn.Module()}[where]
            at.register_buffer("e_score_correction_bias", torch.zeros(4))

    for where in ("block", "experts", "inner"):
        with pytest.raises(NotImplementedError, match="e_score_correction_bias"):
            hf._route_rule(Block(where))
    assert hf._route_rule(Block(None)) == (None, None)


def _described(b, x):
    """The block's result as hf.py describes it: oracle routing, SwiGLU experts, shared expert."""
    from oracle import moe_oracle as O
    from oracle import route_oracle as R
    from promoe_amd import hf
    rule, bias = hf._route_rule(b)
    lg, k = (x @ b.gate.weight.t()).numpy(), int(getattr(b.gate, "top_k", getattr(b, "top_k", 0)))
    if rule is None:
        idx, w = O.topk_route(lg, k, hf._route_mode(b))
        w = w * float(getattr(b.gate, "routed_scaling_factor", 1.0) or 1.0)
    else:
        idx, w = R.route(lg, k, "sigmoid" if rule.scores else "softmax", None if bias is None else bias.numpy(), rule.n_group,
                         rule.topk_group, "top2" if rule.group_value else "max", bool(rule.renorm), rule.scale)
    out, half = torch.zeros_like(x), b.experts.gate_up_proj.shape[1] // 2
    for t in range(len(x)):
        for e, we in zip(idx[t], w[t]):
            gu = b.experts.gate_up_proj[int(e)] @ x[t]
            out[t] += float(we) * (b.experts.down_proj[int(e)] @ (nn.functional.silu(gu[:half]) * gu[half:]))
    sh = hf._shared_expert(b)
    if sh is not None:
        y = sh.down_proj(nn.functional.silu(sh.gate_proj(x)) * sh.up_proj(x))
        gate = getattr(b, "shared_expert_gate", None)
        out += y if gate is None else y * torch.sigmoid(gate(x))
    return out


@pytest.mark.parametrize("name,more", [("DeepseekV3", {}), ("DeepseekV3", dict(n_group=1, topk_group=1, norm_topk_prob=False)),
                                       ("DeepseekV2", dict(topk_method="group_limited_greedy", routed_scaling_factor=2.5)),
                                       ("DeepseekV2", dict(topk_method="greedy")), ("Qwen2Moe", {}), ("Mixtral", {})])
def test_stock_blocks_are_described_as_they_are(name, more):
    """Both sides in fp32 over sums of 64 products; a wrong expert or weight is off by a part of the result."""
    model, blocks = _blocks(name, **more)
    torch.manual_seed(1)
    x = torch.randn(40, 64)
    with torch.no_grad():
        for b in blocks:
            y = b(x[None])
            y = (y[0] if isinstance(y, tuple) else y).reshape(40, 64)
            assert float((_described(b, x) - y).abs().max()) <= 1e-4 * float(y.abs().max())


@pytest.mark.parametrize("case", ["bias on the block", "unknown method"])
def test_a_refused_model_stays_as_it_was(case):
    """The first block could be injected, the last one not: nothing of the model has moved or been dropped when the refusal comes."""
    from promoe_amd import hf
    model, blocks = _blocks("DeepseekV2")
    if case == "unknown method":
        blocks[-1].gate.topk_method = "other"
    else:
        blocks[-1].register_buffer("e_score_correction_bias", torch.zeros(16))
    before = {n: t.clone() for n, t in model.state_dict().items()}
    with pytest.raises(NotImplementedError):
        hf.inject_model(model, device="cpu")
    after = model.state_dict()
    assert list(after) == list(before) and all(torch.equal(after[n], t) and after[n].dtype == t.dtype for n, t in before.items())
    assert not any("forward" in vars(b) for b in blocks)


def test_groups_whose_value_is_unknown_are_refused():
    from promoe_amd import hf
    for name, more in (("Mistral4", dict(norm_topk_prob=True)), ("Mistral4", dict(norm_topk_prob=False))):
        model, blocks = _blocks(name, **more)
        for b in blocks:
            assert hf._route_rule(b) == (None, None)
            with pytest.raises(NotImplementedError, match="2 of 4 groups"):
                hf._route_mode(b)
        model, blocks = _blocks(name, n_group=1, topk_group=1, **more)
        assert hf._route_mode(blocks[0]) == int(more["norm_topk_prob"])


@pytest.mark.parametrize("name,part", [("AXK1", "post_mlp_layernorm"), ("DeepseekV2", "norm")])
def test_a_block_with_further_weights_is_refused(name, part):
    """A norm behind the experts, say: the injected forward would leave it out."""
    from promoe_amd import hf
    model, blocks = _blocks(name)
    if name == "DeepseekV2":
        blocks[-1].act = nn.SiLU()                               # (a part without weights is none)
        hf._check_parts("mlp", blocks[-1])
        blocks[-1].norm = nn.LayerNorm(64)
    with pytest.raises(NotImplementedError, match=part):
        hf.inject_model(model, device="cpu")
    assert blocks[0].experts.gate_up_proj.numel()


def test_biases_below_every_score():
    """Every c below zero: the experts of other groups are still out (not compared as zeros)."""
    model, blocks = _blocks("DeepseekV3")
    torch.manual_seed(2)
    x = torch.randn(40, 64)
    with torch.no_grad():
        for b in blocks:
            b.gate.e_score_correction_bias.add_(-3.0)
            y = b(x[None])
            y = (y[0] if isinstance(y, tuple) else y).reshape(40, 64)
            assert float((_described(b, x) - y).abs().max()) <= 1e-4 * float(y.abs().max())
