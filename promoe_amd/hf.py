"""Model surgery: put the expert cache and the fused MoE layer under a Hugging Face model.

The reference's `inject_model` (reference: src/sparse_llm_cache/utils/__init__.py:147-338) walks a
loaded model, registers every expert's parameters with the loader, moves everything that is not an
expert to the GPU, replaces the experts' storage by slot-backed tensors, and hooks the MoE blocks so
that `report_experts`, the per-expert hooks and the layer hooks run around the model's own expert
loop.  Here the same walk ends in ONE call per MoE block: the block's forward becomes
`moe_forward` (gate, routing, cache hooks, experts, combine and shared expert inside the engine),
and the experts' weights live in pinned host memory as slot images instead of module parameters.

Works on the stock `transformers` sparse blocks that keep their experts in fused tensors
(`experts.gate_up_proj [E, 2I, H]`, `experts.down_proj [E, H, I]`, `gate.weight [E, H]`):
Qwen2-MoE (softmax -> top-k, optional renormalisation, sigmoid-gated shared expert), Mixtral
(softmax -> top-k -> renormalise, which is the softmax over the selected logits) and the DeepSeek
family (DeepSeek-MoE / DeepSeek-V2-Lite: softmax -> greedy top-k without renormalisation, a plain
shared expert `shared_experts` of n_shared_experts * I columns; the reference's metas for it are
utils/common_metas.py:17-41 and 69-94).  Routers with groups of experts (DeepSeek-V2: a group is worth its best expert)
and routers with sigmoid scores and a selection bias (`gate.e_score_correction_bias`; a group is worth its two best) become the
engine's routing rule of the layer (ops.RouteRule); routers and blocks that look like these and are not are refused.  In the DeepSeek models the first decoder layers are dense:
MoE layers are numbered from 0 in model order, so decoder layer i is engine layer
i - first_k_dense_replace (the reference subtracts the same 1, common_metas.py:19-23).  With `fuse_dense` the
dense gated layers run as two launches each (ops.linear_gated, ops.linear).
"""
from __future__ import annotations

import types

import numpy as np
import torch

from . import _lib as L
from . import layout as LY
from . import ops
from . import quant
from .engine import ModuleMeta, PrefetchMngr, PinnedBuffer


def find_moe_blocks(model):
    """[(qualified name, module)] of the sparse MoE blocks, in model order."""
    out = []
    for name, mod in model.named_modules():
        ex = getattr(mod, "experts", None)
        gate = getattr(mod, "gate", None)
        if ex is not None and gate is not None and hasattr(ex, "gate_up_proj") and hasattr(ex, "down_proj") \
                and hasattr(gate, "weight"):
            out.append((name, mod))
    return out


def _check_parts(name, block):
    """Refuses a block with weights that the engine's layer has no place for."""
    known = {"gate", "experts", "shared_expert", "shared_experts", "shared_expert_gate"}
    more = [n for n, m in block.named_children() if n not in known and m.state_dict()]
    if more:
        raise NotImplementedError("block %s of class %s has weights of its own in %s" % (name, type(block).__name__, ", ".join(more)))


def _route_mode(block) -> int:
    gate = block.gate
    if hasattr(gate, "topk_method"):                         # DeepSeek router
        if gate.topk_method != "greedy":
            raise NotImplementedError("DeepSeek routing method %r (only 'greedy' and 'group_limited_greedy' top-k are supported)"
                                      % gate.topk_method)
        return L.ROUTE_SOFTMAX_TOPK
    groups, keep = (next((getattr(o, n) for o in (gate, block) for n in names if getattr(o, n, None) is not None), 1)
                    for names in (("num_group", "n_group"), ("topk_group",)))
    if keep < groups:                                        # (what a group is worth is not to be told from a name)
        raise NotImplementedError("a router of class %s that keeps %d of %d groups of experts" % (type(gate).__name__, keep, groups))
    if hasattr(gate, "norm_topk_prob"):                      # Qwen2-MoE router
        return L.ROUTE_SOFTMAX_TOPK_RENORM if gate.norm_topk_prob else L.ROUTE_SOFTMAX_TOPK
    return L.ROUTE_TOPK_SOFTMAX                              # Mixtral: renormalised top-k of the softmax


def _route_rule(block):
    """(rule, selection bias or None) of a router with groups of experts or sigmoid scores and a selection bias; (None, None)
    for the routers of _route_mode."""
    gate = block.gate

    def find(*names):
        for o in (gate, block):
            for n in names:
                if getattr(o, n, None) is not None:
                    return getattr(o, n)
        raise NotImplementedError("a router of class %s without %s" % (type(gate).__name__, " or ".join(names)))

    bias = getattr(gate, "e_score_correction_bias", None)
    if bias is not None:                                     # scores are sigmoids, the bias balances the choice
        kind = getattr(gate, "scoring_func", None) or getattr(gate, "score_function", None) or "sigmoid"
        if kind != "sigmoid":
            raise NotImplementedError("a selection bias on scores of kind %r (only 'sigmoid' is supported)" % (kind,))
        return ops.RouteRule("sigmoid", int(find("n_group", "num_group")), int(find("topk_group")), "top2",
                             bool(find("norm_topk_prob")), float(find("routed_scaling_factor"))), bias
    if isinstance(block, torch.nn.Module):                   # (on the block or deeper in the gate: routers of other forms, some on softmax)
        other = [n for n in block.state_dict() if n.rsplit(".", 1)[-1] == "e_score_correction_bias"]
        if other:
            raise NotImplementedError("a block of class %s with a selection bias at %s (only one on the gate itself is supported)"
                                      % (type(block).__name__, other[0]))
    if getattr(gate, "topk_method", None) == "group_limited_greedy":
        if getattr(gate, "norm_topk_prob", False):           # (transformers' own router does not divide by the sum; others do)
            raise NotImplementedError("norm_topk_prob with 'group_limited_greedy'")
        return ops.RouteRule("softmax", int(find("num_group", "n_group")), int(find("topk_group")), "max", False,
                             float(find("routed_scaling_factor"))), None
    return None, None


def _activation_of(fn):
    """The name under which ops.linear_gated has a module's activation, from its values; None for any other."""
    # (all over the range, not only where activations bend: clipped ones are others)
    far = torch.tensor([15.0, 20.0, 30.0, 50.0, 1e2, 1e3, 1e4, 1e5, 1e10, 1e30], dtype=torch.float64)
    x = torch.cat([torch.linspace(-12.0, 12.0, 193, dtype=torch.float64), far, -far])
    known = {"silu": torch.nn.functional.silu(x), "gelu": torch.nn.functional.gelu(x),
             "gelu_tanh": torch.nn.functional.gelu(x, approximate="tanh"), "relu": x.relu(), "relu2": x.relu() ** 2}
    try:
        with torch.no_grad():
            y = fn(x.clone())
        return next((n for n, v in known.items() if torch.allclose(y, v, rtol=1e-6, atol=1e-6)), None)
    except Exception:                                        # (one with parameters of another type or device, say)
        return None


class _StandIn(torch.nn.Module):
    """In place of a Linear of the same sizes: column j of the result is the sum of columns j, j + n_out, .. of x, each with a factor."""

    def __init__(self, n_in, n_out, seed, device):
        super().__init__()
        gen = torch.Generator().manual_seed(seed)
        self.in_features, self.out_features, self.rows = n_in, n_out, -(-n_in // n_out)
        self.factor = (1.0 + torch.rand(max(n_in, n_out), dtype=torch.float64, generator=gen)).to(device)
        self.factor[1::2] *= -1.0
        self.weight, self.bias = torch.empty(0, dtype=torch.float64, device=device), None  # (what asks for more of it than its type fails)

    def forward(self, x):
        if self.out_features > self.in_features:
            at = torch.arange(self.out_features, device=x.device) % self.in_features
            return x[..., at] * self.factor
        x = torch.nn.functional.pad(x * self.factor, (0, self.rows * self.out_features - self.in_features))
        return x.unflatten(-1, (self.rows, self.out_features)).sum(-2)


def _is_gated_mlp(mod) -> bool:
    """Does the class's forward compute down(act(gate(x)) * up(x)) and nothing else?  It is run in 64 bits on rows of small and large
    values, over stand-ins for the three products: a factor, a clip or a selection among the columns shows."""
    names = ("gate_proj", "up_proj", "down_proj")
    device = mod.gate_proj.weight.device
    probe = type(mod).__new__(type(mod))
    probe.__dict__.update(mod.__dict__)
    probe.__dict__["_modules"] = dict(mod._modules)
    for i, n in enumerate(names):
        p = getattr(mod, n)
        probe._modules[n] = _StandIn(p.in_features, p.out_features, i, device)
    gen = torch.Generator().manual_seed(7)
    scale = torch.tensor([1e-2, 1.0, 5.0, 30.0, 1e3, 1e5], dtype=torch.float64)[:, None]
    x = (torch.randn(6, mod.gate_proj.in_features, dtype=torch.float64, generator=gen) * scale).reshape(2, 3, -1).to(device)
    try:
        with torch.no_grad():
            y = type(mod).forward(probe, x.clone())
            ref = probe.down_proj(mod.act_fn(probe.gate_proj(x)) * probe.up_proj(x))
        return y.shape == ref.shape and bool(((y - ref).abs() <= 1e-6 * ref.abs().amax(-1, keepdim=True)).all())
    except Exception:                                        # (a forward that needs the weights themselves, or other arguments)
        return False


def _is_plain(m) -> bool:
    """Would calling the module (or function) run its class's forward and nothing else?"""
    return not isinstance(m, torch.nn.Module) or not (m._forward_hooks or m._forward_pre_hooks or "forward" in vars(m))


def find_dense_mlps(model):
    """[(qualified name, module, activation)] of the dense gated feed-forward layers (gate_proj, up_proj, down_proj and act_fn, nothing
    else) that are no part of a sparse block and whose shapes, activation and forward are those of the fused products.  Layers whose
    products are not plain ones (subclasses of Linear: quantised or with adapters; hooks; a forward put in place of the class's) are
    left."""
    inside = {id(m) for _, blk in find_moe_blocks(model) for m in blk.modules()}
    out = []
    for name, mod in model.named_modules():
        parts = [getattr(mod, n, None) for n in ("gate_proj", "up_proj", "down_proj")]
        if id(mod) in inside or not all(type(p) is torch.nn.Linear for p in parts):
            continue
        if not all(_is_plain(m) for m in (*parts, getattr(mod, "act_fn", None))) or "forward" in vars(mod) \
                or set(dict(mod.named_children())) - {"gate_proj", "up_proj", "down_proj", "act_fn"}:
            continue
        g, u, d = parts
        act = _activation_of(getattr(mod, "act_fn", None))
        if act and g.weight.shape == u.weight.shape and d.weight.shape == g.weight.shape[::-1] and d.in_features % 8 == 0 \
                and g.in_features % 8 == 0 and all(p.weight.is_contiguous() and p.weight.data_ptr() % 16 == 0 for p in parts) \
                and _is_gated_mlp(mod):
            out.append((name, mod, act))
    return out


def _fused_mlp_forward(act, act_fn):
    def forward(self, x):
        # (what has been put on or in place of a part since, an adapter or a hook say, has its effect: the class's own forward)
        if self.act_fn is not act_fn or not _is_plain(act_fn) or \
                not all(type(p) is torch.nn.Linear and _is_plain(p) for p in (self.gate_proj, self.up_proj, self.down_proj)):
            return type(self).forward(self, x)
        if x.dtype != self.gate_proj.weight.dtype:           # (autocast brings the types together in the class's own products)
            return type(self).forward(self, x)
        rows = x.detach().reshape(-1, x.shape[-1])
        apart, step = rows.stride()
        if step != 1 or apart % 8 or not rows.shape[1] <= apart < 1 << 21 or rows.data_ptr() % 16:
            rows = rows.clone(memory_format=torch.contiguous_format)
        # (detached, as the engine's own blocks are: nothing here has a gradient)
        w = [None if t is None else t.detach() for p in (self.gate_proj, self.up_proj, self.down_proj) for t in (p.weight, p.bias)]
        h = ops.linear_gated(rows, w[0], w[2], w[1], w[3], act=act)
        return ops.linear(h, w[4], w[5]).reshape(*x.shape[:-1], w[4].shape[0])
    return forward


def _shared_expert(block):
    """The block's always-on expert: Qwen2-MoE calls it shared_expert, the DeepSeek family shared_experts."""
    sh = getattr(block, "shared_expert", None)
    return sh if sh is not None else getattr(block, "shared_experts", None)


def _bf16_bits(t: torch.Tensor) -> np.ndarray:
    return t.detach().to(torch.bfloat16).contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def _expert_image(gate_w, up_w, down_w, H, I, fmt):
    """One SwiGLU expert (torch weights [I,H], [I,H], [H,I]) -> slot image."""
    if fmt == "bf16":
        return LY.pack_expert_bf16(_bf16_bits(gate_w), _bf16_bits(up_w), _bf16_bits(down_w))
    ex = [quant.quantize_int4(w.detach().float().cpu()) for w in (gate_w, up_w, down_w)]
    return LY.pack_expert_int4(ex[0], ex[1], ex[2], H, I)


def inject_model(model, device="cuda:0", fmt: str = "bf16", max_tokens: int = 4096, drop_expert_params: bool = True,
                 fuse_dense: bool = False, **cfg) -> PrefetchMngr:
    """Move the model's dense parts to `device` in bf16, keep its experts in pinned host memory behind the
    slot cache, and route every sparse block through the engine.  Returns the engine (also kept as
    `model._prefetch_mngr`, the attribute the reference attaches, utils/__init__.py:66-70).
    On return torch's current stream is the engine's compute stream: run the model on it.

    fmt "bf16" keeps the experts' weights as they are (rounded to bf16); "int4" quantises them to
    int4-g128 on the way in.  fuse_dense: the dense gated layers (find_dense_mlps) run as two fused launches instead of the
    module's own operations; their intermediate rows are rounded once instead of three times.  Neither they nor the sparse blocks have a
    gradient.  cfg: engine configuration keys (cache_rate, cache_policy, ...).  NotImplementedError: a router or a block that the engine's
    layer cannot stand for (nothing of the model has moved then).
    The shapes must fit the kernels: H and I multiples of 128 (bf16) / 128 and 16 (int4)."""
    if fmt not in ("bf16", "int4"):
        raise ValueError("fmt must be 'bf16' or 'int4'")
    blocks = find_moe_blocks(model)
    if not blocks:
        raise ValueError("the model has no sparse MoE block with fused expert tensors")
    # (every router is read before the first weight moves: a model that is refused stays as it was)
    for name, blk in blocks:
        _check_parts(name, blk)
    rules = [_route_rule(blk) for _, blk in blocks]
    modes = [L.ROUTE_SOFTMAX_TOPK if r is not None else _route_mode(blk) for (r, _), (_, blk) in zip(rules, blocks)]
    b0 = blocks[0][1]
    E, two_i, H = b0.experts.gate_up_proj.shape
    I = two_i // 2
    top_k = int(getattr(b0.gate, "top_k", getattr(b0, "top_k", 0)))
    sh0 = _shared_expert(b0)
    I_sh = sh0.gate_proj.weight.shape[0] if sh0 is not None else 0
    total = LY.bf16_expert_bytes(H, I) if fmt == "bf16" else LY.int4_layout(H, I)["total_bytes"]
    chunks = [("w", 0, total)] if fmt == "bf16" else LY.split_chunks_int4(H, I)

    m = ModuleMeta(len(blocks), E)
    m.init_param_list([c[0] for c in chunks])
    d = {"num_expert_per_token": str(top_k)}
    d.update({a: str(b) for a, b in cfg.items()})
    m.init_from_map(d)
    m.handle_uninited_configs()
    # images first (from the weights as loaded), then the dense parts go to the device
    stage = PinnedBuffer(total * len(blocks) * E)
    shared_imgs = []
    for l, (name, blk) in enumerate(blocks):
        gu, dn = blk.experts.gate_up_proj, blk.experts.down_proj
        if tuple(gu.shape) != (E, 2 * I, H) or tuple(dn.shape) != (E, H, I):
            raise ValueError("block %s differs in shape from the first block" % name)
        # DeepSeek scales the routed experts' sum by a constant; it goes into their down projections (multiplied in
        # fp32, before the one rounding to bf16 / the quantisation of the image)
        # (a layer with a routing rule has it in its weights)
        scale = 1.0 if rules[l][0] is not None else float(getattr(blk.gate, "routed_scaling_factor", 1.0) or 1.0)
        for e in range(E):
            img = _expert_image(gu[e, :I], gu[e, I:], dn[e] if scale == 1.0 else dn[e].detach().float() * scale, H, I, fmt)
            base = (l * E + e) * total
            stage.array[base: base + total] = img
        sh = _shared_expert(blk)
        shared_imgs.append(None if sh is None else
                           _expert_image(sh.gate_proj.weight, sh.up_proj.weight, sh.down_proj.weight, H, I_sh, fmt))
        if drop_expert_params:      # the experts no longer live in the module (nor, later, on the device)
            blk.experts.gate_up_proj = torch.nn.Parameter(torch.empty(0), requires_grad=False)
            blk.experts.down_proj = torch.nn.Parameter(torch.empty(0), requires_grad=False)
            if sh is not None:
                for lin in (sh.gate_proj, sh.up_proj, sh.down_proj):
                    lin.weight = torch.nn.Parameter(torch.empty(0), requires_grad=False)
    # (a selection bias keeps its 32 bits)
    rules = [(r, None if b is None else b.detach().float().to(device)) for r, b in rules]
    model.to(device=device, dtype=torch.bfloat16)
    torch.cuda.set_device(device)
    # a stream of torch's own is handed over as it is; from the legacy default stream (handle 0) the
    # engine makes a private compute stream, and torch is switched onto it, as the reference does
    # (utils/__init__.py:293: torch's current stream := the engine's compute stream)
    pm = PrefetchMngr(m, backend=L.BACKEND_HIP, compute_stream=torch.cuda.current_stream().cuda_stream)
    pm._keep.append(stage)
    if pm.compute_stream != torch.cuda.current_stream().cuda_stream:
        prev = torch.cuda.current_stream()
        torch.cuda.synchronize()
        torch.cuda.set_stream(torch.cuda.ExternalStream(pm.compute_stream, device=device))
        engine_close = pm.close

        def close():  # the stream dies with the engine: give torch its own stream back first
            torch.cuda.synchronize()
            torch.cuda.set_stream(prev)
            engine_close()
        pm.close = close
    for l in range(len(blocks)):
        for e in range(E):
            base = (l * E + e) * total
            for cname, off, n in chunks:
                pm.add_one_expert_param(stage.array[base + off: base + off + n], l, e, cname)
    pm.init_gpu_mem_buffer()
    for l, (name, blk) in enumerate(blocks):
        gw = blk.gate.weight.detach().to(torch.bfloat16)
        sg = getattr(blk, "shared_expert_gate", None)
        if sg is not None:
            gw = torch.cat([gw, sg.weight.detach().to(torch.bfloat16).reshape(1, H)])
        sh = None if shared_imgs[l] is None else torch.from_numpy(np.ascontiguousarray(shared_imgs[l])).to(device)
        pm.set_layer(l, H, I, I_sh, top_k, modes[l], gw.contiguous(), None, sh, shared_gated=sg is not None,
                     fmt=L.FMT_BF16 if fmt == "bf16" else L.FMT_INT4_G128, rule=rules[l][0], select_bias=rules[l][1])
    pm.forward_prepare(max_tokens)
    pm.launch_thread()

    def make_forward(layer_id):
        def forward(self, hidden_states):
            shape = hidden_states.shape
            x = hidden_states.reshape(-1, shape[-1]).to(torch.bfloat16).contiguous()
            if x.shape[0] > max_tokens:
                raise ValueError("%d tokens in one forward, the engine was prepared for %d" % (x.shape[0], max_tokens))
            y = pm.forward(layer_id, x)
            return y.reshape(shape).to(hidden_states.dtype)
        return forward

    for l, (name, blk) in enumerate(blocks):
        blk._layer_id = l                                   # the reference's metadata attribute (utils/__init__.py:25-31)
        blk.forward = types.MethodType(make_forward(l), blk)
    if fuse_dense:
        for _, mod, act in find_dense_mlps(model):
            mod.forward = types.MethodType(_fused_mlp_forward(act, mod.act_fn), mod)
    model._prefetch_mngr = pm
    return pm
