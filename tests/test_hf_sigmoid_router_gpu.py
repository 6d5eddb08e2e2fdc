"""A stock transformers model whose router has sigmoid scores, a selection bias and groups worth two experts: its sparse blocks through
the engine against the same blocks run by transformers itself, and the model as a whole."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(seed, **kw):
    transformers = pytest.importorskip("transformers")
    if not hasattr(transformers, "DeepseekV3ForCausalLM"):
        pytest.skip("this transformers has no such model")
    d = dict(vocab_size=128, hidden_size=256, intermediate_size=520, moe_intermediate_size=128, num_hidden_layers=3, num_attention_heads=4,
             num_key_value_heads=4, n_shared_experts=1, n_routed_experts=32, num_experts_per_tok=4, first_k_dense_replace=1, kv_lora_rank=32,
             q_lora_rank=None, qk_rope_head_dim=16, qk_nope_head_dim=32, v_head_dim=32, n_group=8, topk_group=3, norm_topk_prob=True,
             routed_scaling_factor=2.5, max_position_embeddings=128)
    d.update(kw)
    torch.manual_seed(seed)
    model = transformers.DeepseekV3ForCausalLM(transformers.DeepseekV3Config(**d)).eval()
    with torch.no_grad():
        for layer in model.model.layers[1:]:
            layer.mlp.gate.weight.copy_(torch.randn_like(layer.mlp.gate.weight) * 0.1)
            # (a balance bias moves choices, it does not take every score below zero)
            layer.mlp.gate.e_score_correction_bias.copy_(torch.randn(layer.mlp.gate.weight.shape[0]) * 0.05)
    return model


@pytest.mark.parametrize("kw", [dict(), dict(norm_topk_prob=False, routed_scaling_factor=1.0), dict(n_group=1, topk_group=1)])
def test_blocks_of_a_stock_model(cuda, kw):
    """Outputs off by the roundings of bf16 rows between the products, as in the layer's other tests; choices those of the rule."""
    from oracle import route_oracle as R
    from promoe_amd import hf
    model = _model(3, **kw)
    ref = copy.deepcopy(model).to(device=cuda, dtype=torch.bfloat16)
    cfg = model.config
    # (transformers rounds the bias to bf16 with the rest of the model; the engine keeps its 32 bits)
    for layer in model.model.layers[1:]:
        b = layer.mlp.gate.e_score_correction_bias
        b.copy_(b.to(torch.bfloat16).float())
    pm = hf.inject_model(model, device=cuda, max_tokens=128, cache_rate=0.5, cache_policy="lru", fuse_dense=True)
    try:
        for T in (1, 5, 40, 100):
            for l in (0, 1):
                print(f"case hf_sigmoid_stock {kw} T={T} layer={l}", flush=True)
                gen = torch.Generator(device=cuda).manual_seed(10 * T + l)
                x = torch.randn(1, T, 256, device=cuda, generator=gen).to(torch.bfloat16)
                a, b = ref.model.layers[l + 1].mlp, model.model.layers[l + 1].mlp
                with torch.no_grad():
                    ya, yb = a(x), b(x)
                lg = (x[0].double().cpu() @ a.gate.weight.detach().double().cpu().t()).float().numpy()
                idx = R.route(lg, cfg.num_experts_per_tok, "sigmoid", a.gate.e_score_correction_bias.float().cpu().numpy(), cfg.n_group,
                              cfg.topk_group, "top2")[0]
                assert np.array_equal(pm.last_routing_idx(T, cfg.num_experts_per_tok), idx)
                assert float((ya.float() - yb.float()).abs().max()) <= 2e-2 * float(ya.float().abs().max())
        ids = torch.randint(0, 128, (1, 12), device=cuda)
        with torch.no_grad():
            out = model(ids, use_cache=True)
            out = model(out.logits[:, -1:].argmax(-1), past_key_values=out.past_key_values, use_cache=True)
        assert torch.isfinite(out.logits).all()
    finally:
        pm.close()
