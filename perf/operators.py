"""Operators beside the expert layers: routers with groups and a selection bias, and the products of dense feed-forward layers.

  route      scores (sigmoid, or softmax over all experts), a selection bias, groups of experts, top-k, weights
  dispatch   the same and the stable dispatch behind it, for decode batches
  linear     act(x W^T + b) + residual
  gated      act(x Wg^T + bg) * (x Wu^T + bu)

Sizes: experts, choices, hidden and intermediate sizes of the configured MoE shapes (2048 x 1408, 60 and 64 experts, 4096 x
14336, 3584 x 2560) and the dense layers between such blocks, or generic ones.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _route(name, op, T, E, k, scores, bias, n_group=1, topk_group=1, group_value="max", renorm=False, scale=1.0, extra=0):
    """extra: columns behind the experts' in a row of logits (the shared expert's gate logit)"""
    c = dict(op=op, T=T, E=E, k=k, scores=scores, bias=bias, n_group=n_group, topk_group=topk_group, group_value=group_value,
             renorm=renorm, scale=scale, extra=extra)
    return dict(c, name=name) if name else c


def _product(name, op, M, N, K, dtype, act="none", bias=False, residual=False, out="same"):
    """out "fp32": sums leave in fp32 (partial rows, scores); "same": in the type of x"""
    c = dict(op=op, M=M, N=N, K=K, dtype=dtype, act=act, bias=bias, residual=residual, out=out)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a sequence being decoded: one row of 64 logits, sigmoid scores with a balance bias; latency is all there is
        _route("route 1 x 64 sigmoid", "route", 1, 64, 6, "sigmoid", True, renorm=True),
        # a prompt of odd length through a gated layer of 60 experts in 6 groups: rows of 61 logits
        _route("route 379 x 60 groups", "route", 379, 60, 4, "softmax", False, 6, 3, "max", extra=1),
        # a large batch of prompts, 256 experts in 8 groups with a balance bias
        _route("route 32768 x 256 groups", "route", 32768, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5),
        # decode steps: routing and the unit list for the expert launch, one sequence and a serving batch
        _route("dispatch 1 x 64", "dispatch", 1, 64, 6, "softmax", False, 8, 3, "max"),
        _route("dispatch 33 x 256", "dispatch", 33, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5),
        # second half of a dense layer in a decode step: 45 MB of weights for one row
        _product("linear 1 x 2048 x 10944", "linear", 1, 2048, 10944, "bf16", residual=True),
        # a serving batch through a projection with a bias
        _product("linear 24 x 4096 x 4096", "linear", 24, 4096, 4096, "fp16", bias=True),
        # odd rows and columns, everything in the epilogue
        _product("linear 379 x 1409 x 2048", "linear", 379, 1409, 2048, "fp16", "gelu", True, True),
        # a full prompt through the second half of a wide dense layer
        _product("linear 4096 x 4096 x 14336", "linear", 4096, 4096, 14336, "bf16", residual=True),
        # first half of a dense layer in a decode step: 90 MB of weights for one row
        _product("gated 1 x 10944 x 2048", "gated", 1, 10944, 2048, "bf16", "silu"),
        # a short prompt of odd length: neither streaming nor a full chip of tiles
        _product("gated 251 x 2560 x 3584", "gated", 251, 2560, 3584, "fp16", "gelu_tanh", True),
        # a full prompt through the first half of a wide dense layer, the largest call
        _product("gated 4096 x 14336 x 4096", "gated", 4096, 14336, 4096, "bf16", "silu"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["route", "dispatch", "linear", "linear", "gated", "gated"])
    if op in ("route", "dispatch"):
        n_group = rng.choice([1, 1, 2, 4, 6, 8])
        size = rng.randint(2 if n_group > 1 else 8, 256 // n_group)
        E = n_group * size
        topk_group = rng.randint((n_group + 1) // 2, n_group)
        k = rng.randint(1, min(8, topk_group * size))
        T = _log(rng, 1, 32768) if op == "route" else _log(rng, 1, 64)
        return _route(None, op, T, E, k, rng.choice(["sigmoid", "softmax"]), rng.random() < 0.6, n_group, topk_group,
                      rng.choice(["max", "top2"]), rng.random() < 0.5, rng.choice([1.0, 2.5, 16.0]), rng.choice([0, 1]))
    most = 4096 * 14336 * 4096 * (1 if op == "gated" else 2)
    while True:
        M, N, K = _log(rng, 1, 4096), _log(rng, 64, 16384), 8 * _log(rng, 32, 1792)
        if M * N * K <= most:
            break
    dtype = rng.choice(sorted(TYPES))
    bias = rng.random() < 0.5
    if op == "gated":
        return _product(None, op, M, N, K, dtype, rng.choice(["silu", "gelu", "gelu_tanh"]), bias)
    return _product(None, op, M, N, K, dtype, rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu", "relu2"]), bias,
                    rng.random() < 0.5, rng.choice(["same", "same", "same", "fp32"]))


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, std, dtype=torch.float32):
        return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)

    if case["op"] in ("route", "dispatch"):
        # logits of a gate over normalised hidden states; a balance bias as it stands after some training
        rows = normal((case["T"], case["E"] + case["extra"]), 1.2)
        return {"logits": rows[:, :case["E"]], "bias": normal((case["E"],), 0.05) if case["bias"] else None}
    M, N, K, t = case["M"], case["N"], case["K"], TYPES[case["dtype"]]
    s = {"x": normal((M, K), 1.0, t)}
    parts = ("gate", "up") if case["op"] == "gated" else ("w",)
    for p in parts:
        s[p] = normal((N, K), 0.02, t)
        s["b_" + p] = normal((N,), 0.1, t) if case["bias"] else None
    if case["op"] == "linear":
        s["residual"] = normal((M, N), 1.0, t) if case["residual"] else None
    return s


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own and case["op"] in ("route", "dispatch"):
        from promoe_amd import ops
        state["rule"] = ops.RouteRule(case["scores"], case["n_group"], case["topk_group"], case["group_value"], case["renorm"],
                                      case["scale"])
    return state


def _run_own(state):
    from promoe_amd import ops
    case = state["case"]
    if case["op"] == "route":
        return ops.group_topk(state["logits"], case["k"], state["rule"], state["bias"])
    if case["op"] == "dispatch":
        idx, w, d = ops.group_topk_dispatch(state["logits"], case["k"], state["rule"], state["bias"])
        return idx, w, d.counts, d.offsets, d.sorted_pair, d.pos_of_pair, d.sorted_tok, d.units, d.n_active, d.active_ids
    if case["op"] == "linear":
        return ops.linear(state["x"], state["w"], state["b_w"], act=case["act"], residual=state["residual"],
                          out_dtype=torch.float32 if case["out"] == "fp32" else None)
    return ops.linear_gated(state["x"], state["gate"], state["up"], state["b_gate"], state["b_up"], act=case["act"])


def _choose(case, logits, bias):
    """idx [T, k] int32 and w [T, k] fp32; scores and comparisons in 64 bits"""
    T, E, G, k = case["T"], case["E"], case["n_group"], case["k"]
    l = logits.double()
    if case["scores"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
    else:
        e = torch.exp(l - l.max(dim=1, keepdim=True).values)
        s = e / e.sum(dim=1, keepdim=True)
    c = s if bias is None else s + bias.double()
    if G > 1:
        g = c.view(T, G, E // G)
        best = torch.sort(g, dim=2, descending=True).values
        v = best[:, :, 0] + best[:, :, 1] if case["group_value"] == "top2" else best[:, :, 0]
        order = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :case["topk_group"]]
        kept = torch.zeros(T, G, dtype=torch.bool, device=l.device).scatter_(1, order, True)
        c = torch.where(kept[:, :, None], g, -math.inf).reshape(T, E)
    idx = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :k]
    w = torch.gather(s, 1, idx)
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return idx.int(), (w * case["scale"]).float()


def _dispatch(idx, E):
    """The pairs (token, choice) in stable order of their experts, and the experts in use."""
    T, k = idx.shape
    P, dev = T * k, idx.device
    flat = idx.reshape(-1).long()
    counts = (flat[:, None] == torch.arange(E, device=dev)).sum(dim=0)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), torch.cumsum(counts, 0)])
    pairs = torch.sort(flat, stable=True).indices
    pos = torch.empty_like(pairs)
    pos[pairs] = torch.arange(P, device=dev)
    most = min(E, P)
    used = counts > 0
    n_active = used.sum().reshape(1)
    slot = torch.where(used, torch.cumsum(used, 0) - 1, most)     # an expert not in use goes behind the last place
    units = torch.zeros(most + 1, 4, dtype=torch.int64, device=dev)
    units[:, 0] = -1
    rows = torch.stack([torch.arange(E, device=dev), counts, offsets[:-1], torch.zeros_like(counts)], dim=1)
    units[slot] = rows
    ids = torch.full((most + 1,), -1, dtype=torch.int64, device=dev)
    ids[slot] = torch.arange(E, device=dev)
    return (counts.int(), offsets.int(), pairs.int(), pos.int(), (pairs // k).int(), units[:most].int(), n_active.int(),
            ids[:most])


def _act(name, v):
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "relu":
        return torch.clamp(v, min=0.0)
    if name == "relu2":
        r = torch.clamp(v, min=0.0)
        return r * r
    return v


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] in ("route", "dispatch"):
        idx, w = _choose(case, state["logits"], state["bias"])
        return (idx, w) + (_dispatch(idx, case["E"]) if case["op"] == "dispatch" else ())
    x = state["x"].float()

    def product(w, b):
        v = x @ w.float().t()
        return v if b is None else v + b.float()

    if case["op"] == "gated":
        y = _act(case["act"], product(state["gate"], state["b_gate"])) * product(state["up"], state["b_up"])
        return y.to(state["x"].dtype)
    y = _act(case["act"], product(state["w"], state["b_w"]))
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y if case["out"] == "fp32" else y.to(state["x"].dtype)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("route", "dispatch"):
        return _exact_route(case, s)
    x = s["x"].double()
    erf, tanh = torch.special.erf, torch.tanh

    def half(name):
        v = torch.empty(case["M"], case["N"], dtype=torch.float64, device="cuda")
        for j in range(0, case["N"], 2048):
            v[:, j: j + 2048] = torch.mm(x, s[name][j: j + 2048].double().t().contiguous())
        if case["bias"]:
            v += s["b_" + name].double()
        return v

    fn = {"none": lambda v: v, "relu": lambda v: v * (v > 0), "relu2": lambda v: v * v * (v > 0),
          "silu": lambda v: v * torch.special.expit(v), "gelu": lambda v: v * (1 + erf(v / math.sqrt(2))) / 2,
          "gelu_tanh": lambda v: v * (1 + tanh((v + 0.044715 * v ** 3) * math.sqrt(2 / math.pi))) / 2}[case["act"]]
    if case["op"] == "gated":
        return fn(half("gate")) * half("up")
    y = fn(half("w"))
    return y if s["residual"] is None else y + s["residual"].double()


def _exact_route(case, s):
    """Row by row selection by repeated maxima; the whole numbers have no value but the plain one's, so they are left out"""
    T, E, G, k = case["T"], case["E"], case["n_group"], case["k"]
    l = s["logits"].double()
    p = torch.special.expit(l) if case["scores"] == "sigmoid" else torch.softmax(l, dim=1)
    c = p.clone() if s["bias"] is None else p + s["bias"].double()
    rows = torch.arange(T, device=l.device)
    if G > 1:
        left, value = c.reshape(T * G, E // G).clone(), 0.0
        for _ in range(2 if case["group_value"] == "top2" else 1):
            m, at = left.max(dim=1)
            value = value + m
            left[torch.arange(T * G, device=l.device), at] = -math.inf
        value = value.reshape(T, G)
        out = torch.ones(T, G, dtype=torch.bool, device=l.device)
        for _ in range(case["topk_group"]):
            at = value.max(dim=1).indices
            out[rows, at] = False
            value[rows, at] = -math.inf
        c[out.repeat_interleave(E // G, dim=1)] = -math.inf
    w = torch.empty(T, k, dtype=torch.float64, device=l.device)
    for j in range(k):
        at = c.max(dim=1).indices
        w[:, j] = p[rows, at]
        c[rows, at] = -math.inf
    if case["renorm"]:
        w /= w.sum(dim=1, keepdim=True)
    w *= case["scale"]
    return (None, w) + ((None,) * 8 if case["op"] == "dispatch" else ())


def work(case):
    if case["op"] in ("route", "dispatch"):
        T, E, k = case["T"], case["E"], case["k"]
        nbytes = T * E * 4 + T * k * 8 + (E * 4 if case["bias"] else 0)
        if case["op"] == "dispatch":
            nbytes += (2 * E + 1) * 4 + 3 * T * k * 4 + min(E, T * k) * 24 + 4
        # a score is an exponential, a division and the sums: about ten operations
        return {"bytes": nbytes, "flops": 10.0 * T * E}
    M, N, K = case["M"], case["N"], case["K"]
    mats = 2 if case["op"] == "gated" else 1
    nbytes = 2 * (M * K + mats * N * K) + (4 if case["out"] == "fp32" else 2) * M * N
    nbytes += 2 * mats * N if case["bias"] else 0
    nbytes += 2 * M * N if case["residual"] else 0
    return {"bytes": nbytes, "flops": 2.0 * mats * M * N * K}
