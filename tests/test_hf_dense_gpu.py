"""A stock transformers model with a group-limited router, and dense layers as fused products, through the engine, against the same
model run by transformers itself; a router with sigmoid scores and a selection bias on a block that presents one."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(seed, dense=1, **kw):
    from transformers import DeepseekV2Config, DeepseekV2ForCausalLM
    d = dict(vocab_size=128, hidden_size=256, intermediate_size=520, moe_intermediate_size=128, num_hidden_layers=3,
             num_attention_heads=4, num_key_value_heads=4, n_shared_experts=2, n_routed_experts=16, num_experts_per_tok=4,
             first_k_dense_replace=dense, kv_lora_rank=32, q_lora_rank=None, qk_rope_head_dim=16, qk_nope_head_dim=32, v_head_dim=32,
             head_dim=16, topk_method="group_limited_greedy", n_group=4, topk_group=2, routed_scaling_factor=2.5,
             max_position_embeddings=128)
    d.update(kw)
    torch.manual_seed(seed)
    return DeepseekV2ForCausalLM(DeepseekV2Config(**d)).eval()


def _rel(a, b):
    return float((a.float() - b.float()).abs().max() / b.float().abs().max())


@pytest.mark.parametrize("fuse", [False, True])
@pytest.mark.parametrize("dense", [1, 2])
def test_group_limited_model_through_the_engine(cuda, fuse, dense):
    """Prefill and cached decode, with the dense layers as the module has them and fused."""
    print(f"case hf_group_limited fuse={fuse} dense={dense}", flush=True)
    from promoe_amd import hf
    model = _model(5, dense)
    ref = copy.deepcopy(model).to(device=cuda, dtype=torch.bfloat16)
    assert [n for n, _, _ in hf.find_dense_mlps(model)] == ["model.layers.%d.mlp" % i for i in range(dense)]
    calls = []
    from promoe_amd import ops
    gated = ops.linear_gated
    pm = hf.inject_model(model, device=cuda, max_tokens=64, fuse_dense=fuse, cache_rate=0.5, cache_policy="lru")
    try:
        ops.linear_gated = lambda *a, **k: (calls.append(1), gated(*a, **k))[1]
        ids = torch.randint(0, 128, (1, 12), device=cuda)
        with torch.no_grad():
            a, b = ref(ids, use_cache=True), model(ids, use_cache=True)
            errs = [_rel(b.logits, a.logits)]
            pa, pb = a.past_key_values, b.past_key_values
            tok = a.logits[:, -1:].argmax(-1)
            for _ in range(3):
                a, b = ref(tok, past_key_values=pa, use_cache=True), model(tok, past_key_values=pb, use_cache=True)
                errs.append(_rel(b.logits, a.logits))
                pa, pb = a.past_key_values, b.past_key_values
                tok = a.logits[:, -1:].argmax(-1)
        torch.cuda.synchronize()
        print("  logits max-rel-err per forward:", ["%.3e" % e for e in errs], flush=True)
        assert max(errs) <= 3e-2
        assert len(calls) == (4 * dense if fuse else 0)
    finally:
        ops.linear_gated = gated
        pm.close()


def test_fused_dense_layer_of_a_model(cuda):
    """The layer alone, fused, against its formula in 64 bits on its bf16 weights: intermediate rounded once (2^-8 of a value), then
    the result (2^-8)."""
    print("case hf_fused_mlp", flush=True)
    from promoe_amd import hf
    model = _model(6)
    pm = hf.inject_model(model, device=cuda, max_tokens=64, fuse_dense=True)
    try:
        mlp = model.model.layers[0].mlp
        gen = torch.Generator(device=cuda).manual_seed(1)
        x = torch.randn(2, 7, 256, device=cuda, generator=gen).to(torch.bfloat16)
        y = mlp(x)
        assert y.shape == x.shape and y.dtype == torch.bfloat16 and not y.requires_grad
        wg, wu, wd = (p.weight.detach().double() for p in (mlp.gate_proj, mlp.up_proj, mlp.down_proj))
        xd = x.double().reshape(-1, 256)
        g = torch.mm(xd, wg.t().contiguous())
        h = g / (1 + torch.exp(-g)) * torch.mm(xd, wu.t().contiguous())
        ref = torch.mm(h, wd.t().contiguous())
        tol = 2.0 ** -8 * torch.mm(h.abs(), wd.abs().t().contiguous()) * 1.01 + 2.0 ** -8 * 1.01 * ref.abs() + 1e-6
        assert ((y.double().reshape(-1, 256) - ref).abs() <= tol).all()
    finally:
        pm.close()


def test_sigmoid_router_with_a_selection_bias(cuda):
    """A block that presents such a router (transformers' stock names) routes as the rule says."""
    print("case hf_sigmoid_router", flush=True)
    from oracle import route_oracle as R
    from promoe_amd import hf
    model = _model(7)
    for i in (1, 2):
        gate = model.model.layers[i].mlp.gate
        gate.register_buffer("e_score_correction_bias", torch.linspace(-0.2, 0.2, 16).roll(3 * i))
        gate.n_group, gate.norm_topk_prob = 4, True
    weights = [model.model.layers[i].mlp.gate.weight.detach().to(torch.bfloat16).float().numpy() for i in (1, 2)]
    bias = [model.model.layers[i].mlp.gate.e_score_correction_bias.numpy().copy() for i in (1, 2)]
    pm = hf.inject_model(model, device=cuda, max_tokens=64)
    try:
        from oracle import moe_oracle as O
        for l in (0, 1):
            for T in (1, 5, 40):
                x = O.synth_acts(T, 256, seed=T + l)
                pm.forward(l, torch.from_numpy(x).to(torch.bfloat16).to(cuda))
                idx = pm.last_routing_idx(T, 4)
                ref = R.route(O.gate_logits_ordered(x, weights[l]), 4, "sigmoid", bias[l], 4, 2, "top2", True, 2.5)[0]
                assert np.array_equal(idx, ref), (l, T)
    finally:
        pm.close()


def test_a_router_that_lacks_what_a_rule_needs_is_refused():
    from promoe_amd import hf
    model = _model(8)
    gate = model.model.layers[1].mlp.gate
    gate.register_buffer("e_score_correction_bias", torch.zeros(16))
    with pytest.raises(NotImplementedError, match="norm_topk_prob"):
        hf._route_rule(model.model.layers[1].mlp)
    assert hf._route_rule(model.model.layers[2].mlp)[0].n_group == 4
