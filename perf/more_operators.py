"""Experts and dense layers with weights in microscaled 4-bit floating point, and the way of the tokens to the experts and back.

  quantize   rows of 16 or 32 bits -> 4-bit codes with one power of two per 32 of them, and back
  linear     act(x W^T + b) + residual, W in 4 bits; x in 16 bits, or quantised in the call ("x": "mx4")
  gated      act(x Wg^T + bg) * (x Wu^T + bu), the same
  experts    these two products of every expert with the rows of its tokens, in one call
  sort       rows of the tokens in the order of their experts (a token's row once per choice), and its gradient
  unsort     the experts' rows back to the tokens, weighted and summed, and its gradients

A block of 32 values has the scale 2^(floor(log2 of its largest magnitude) - 2), at least 2^-127; a code is the nearest of
0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives to value / scale, of two as near the one with the even code, 6 beyond.

Sizes: experts, choices, hidden and intermediate sizes of the configured MoE shapes (2048 x 1408, 60 and 64 experts, 4096 x
14336 with 8, 3584 x 2560 with 64) and the dense layers between such blocks, or generic ones.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _quantize(name, M, K, dtype):
    c = dict(op="quantize", M=M, K=K, dtype=dtype)
    return dict(c, name=name) if name else c


def _product(name, op, M, N, K, x, dtype="bf16", act="none", bias=False, residual=False, out="same"):
    """x "mx4": rows of `dtype` are quantised in the call; "16": they stay as they are.  out "fp32", or "same" as `dtype`"""
    c = dict(op=op, M=M, N=N, K=K, x=x, dtype=dtype, act=act, bias=bias, residual=residual, out=out)
    return dict(c, name=name) if name else c


def _experts(name, T, E, k, N, K, gated, x, dtype="bf16", act="silu", bias=False):
    """gated: first half of the experts, from the tokens' rows; otherwise the second half, from rows in the experts' order"""
    c = dict(op="experts", T=T, E=E, k=k, N=N, K=K, gated=gated, x=x, dtype=dtype, act=act if gated else "none", bias=bias)
    return dict(c, name=name) if name else c


def _move(name, op, T, H, k, E, dtype, grad, left=0.0):
    """grad: the gradients as well (a training step); left: share of choices that belong to experts elsewhere"""
    c = dict(op=op, T=T, H=H, k=k, E=E, dtype=dtype, grad=grad, left=left)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the hidden state of one sequence, on its way to a product in 4 bits: the smallest call
        _quantize("quantize 1 x 2048", 1, 2048, "bf16"),
        # the rows between the two halves of a wide dense layer, a full prompt
        _quantize("quantize 4096 x 14336", 4096, 14336, "bf16"),
        # second half of a dense layer in a decode step: 12 MB of weights for one row
        _product("linear 1 x 2048 x 10944", "linear", 1, 2048, 10944, "16", residual=True),
        # odd rows and columns, everything in the epilogue, a short prompt that is not to be rounded
        _product("linear 379 x 1409 x 2048", "linear", 379, 1409, 2048, "16", "fp16", "gelu", True, True),
        # a full prompt through the second half of a wide dense layer, both operands in 4 bits
        _product("linear 4096 x 4096 x 14336", "linear", 4096, 4096, 14336, "mx4", residual=True),
        # first half of the experts in a decode step: six experts of 64 for one row
        _experts("experts 1 of 64 top 6 gated", 1, 64, 6, 1408, 2048, True, "16"),
        # a full prompt through the first half of 64 narrow experts: about 192 rows each
        _experts("experts 2048 of 64 top 6 gated", 2048, 64, 6, 1408, 2048, True, "mx4"),
        # a full prompt through the second half of 8 wide experts, the largest call
        _experts("experts 4096 of 8 top 2", 4096, 8, 2, 4096, 14336, False, "mx4"),
        # a serving batch to its experts
        _move("sort 33 x 3584 top 8", "sort", 33, 3584, 8, 64, "bf16", False),
        # a training step: rows of a batch to the experts, and the gradient of the hidden states
        _move("sort 4096 x 2048 top 6 trained", "sort", 4096, 2048, 6, 64, "bf16", True),
        # a serving batch of odd length back from its experts, a part of which are elsewhere
        _move("unsort 37 x 3584 top 8", "unsort", 37, 3584, 8, 64, "fp16", False, 0.25),
        # the experts' rows of a training batch back, and the gradients of the rows and of the routing weights
        _move("unsort 4096 x 2048 top 6 trained", "unsort", 4096, 2048, 6, 64, "bf16", True),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


MOST = 8192 * 4096 * 14336  # products of the largest listed case


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "gated", "experts", "experts", "sort", "unsort"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "quantize":
        return _quantize(None, _log(rng, 1, 4096), 32 * _log(rng, 1, 448), rng.choice(["bf16", "fp16", "fp32"]))
    if op in ("sort", "unsort"):
        return _move(None, op, _log(rng, 1, 4096), 8 * _log(rng, 8, 448), rng.randint(1, 8), rng.choice([8, 60, 64, 256]), dtype,
                     rng.random() < 0.5, rng.choice([0.0, 0.0, 0.25]))
    x = rng.choice(["mx4", "16"])
    if op == "experts":
        gated = rng.random() < 0.5
        while True:
            T, E = _log(rng, 1, 4096), rng.choice([8, 16, 60, 64])
            k = rng.randint(1, min(E, 8))
            N, K = _log(rng, 256, 14336), 32 * _log(rng, 8, 448)
            # (the matrices of all experts are in hand: as many as the configured layers have, at most)
            if T * k * N * K * (2 if gated else 1) <= MOST and E * N * K * (2 if gated else 1) <= 1 << 29:
                break
        return _experts(None, T, E, k, N, K, gated, x, dtype, rng.choice(["silu", "gelu", "gelu_tanh"]), rng.random() < 0.3)
    while True:
        M, N, K = _log(rng, 1, 4096), _log(rng, 64, 16384), 32 * _log(rng, 8, 448)
        if M * N * K * (2 if op == "gated" else 1) <= MOST:
            break
    bias = rng.random() < 0.5
    if op == "gated":
        return _product(None, op, M, N, K, x, dtype, rng.choice(["silu", "gelu", "gelu_tanh"]), bias)
    return _product(None, op, M, N, K, x, dtype, rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu", "relu2"]), bias,
                    rng.random() < 0.5, rng.choice(["same", "same", "same", "fp32"]))


GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _scale_bits(b):
    """The biased exponent of the scale of each block of the last dimension, int32"""
    top = (b.abs().amax(-1).view(torch.int32) >> 23) & 255
    return torch.where(top == 255, top, torch.clamp(top - 2, min=0))


def _steps(b, bits):
    """b / scale rounded to the grid (fp32)"""
    v = torch.ldexp(b, (127 - bits)[..., None])
    r = v.abs()
    q = torch.where(r < 2, torch.round(r * 2) / 2, torch.where(r < 4, torch.round(r), torch.round(r / 2) * 2))
    return torch.clamp(q, max=6.0) * torch.sign(v)


def _rounded(x):
    """The values that the rows of x stand for once they are quantised (fp32)"""
    b = x.float().unflatten(-1, (-1, 32))
    bits = _scale_bits(b)
    return torch.ldexp(_steps(b, bits), (bits - 127)[..., None]).flatten(-2)


def _packed(x):
    """codes uint8 [..., K / 2] (the even column in the low half) and scales uint8 [..., K / 32] of x"""
    b = x.float().unflatten(-1, (-1, 32))
    bits = _scale_bits(b)
    q = _steps(b, bits)
    grid = torch.tensor(GRID, device=x.device)
    c = (torch.bucketize(q.abs(), grid).to(torch.uint8) + 8 * (q < 0).to(torch.uint8)).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), bits.to(torch.uint8)


def _unpacked(w):
    """fp32 values of (codes, scales)"""
    codes, scales = w
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).int()
    v = grid[c].unflatten(-1, (-1, 32))
    return torch.ldexp(v, (scales.int() - 127)[..., None]).flatten(-2)


def _routing(case, gen):
    """Choices of each token (-1: of an expert elsewhere), their weights, and the stable order of the pairs by expert"""
    T, k, E = case["T"], case["k"], case["E"]
    scores = torch.randn(T, E, device="cuda", generator=gen)
    top = torch.topk(scores, k, dim=1)
    idx, w = top.indices.int(), torch.softmax(top.values, dim=1)
    if case.get("left"):
        idx[torch.rand(T, k, device="cuda", generator=gen) < case["left"]] = -1
    flat = torch.where(idx < 0, E, idx).reshape(-1).long()
    order = torch.sort(flat, stable=True).indices
    pos = torch.empty_like(order)
    pos[order] = torch.arange(T * k, device="cuda")
    counts = torch.bincount(flat, minlength=E + 1)[:E]
    return {"idx": idx, "weights": w, "order": order, "pos": pos, "counts": counts, "here": int(counts.sum()), "sizes": counts.tolist()}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, op = TYPES[case["dtype"]], case["op"]

    def normal(shape, std, dtype=torch.float32):
        return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)

    def matrices(E, N, K):
        """E matrices (None: one) as codes and scales, quantised a few at a time"""
        if E is None:
            return _packed(normal((N, K), 0.02))
        parts = [_packed(normal((1, N, K), 0.02)) for _ in range(E)]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])

    if op == "quantize":
        # hidden states: some columns are always far larger than the others
        far = torch.exp(torch.randn(case["K"], device="cuda", generator=gen))
        return {"x": (normal((case["M"], case["K"]), 1.0) * far).to(t)}
    if op in ("sort", "unsort"):
        s = _routing(case, gen)
        rows = case["T"] if op == "sort" else case["T"] * case["k"]
        s["x"] = normal((rows, case["H"]), 1.0, t)
        s["g"] = normal((case["T"] * case["k"] if op == "sort" else case["T"], case["H"]), 1e-2, t) if case["grad"] else None
        return s
    s, N, K, E = {}, case["N"], case["K"], None
    if op == "experts":
        E = case["E"]
        s = _routing(case, gen)
    gated = case["gated"] if op == "experts" else op == "gated"
    M = case["M"] if op != "experts" else case["T"] if gated else case["T"] * case["k"]
    s["x"] = normal((M, K), 1.0, t)
    for p in ("gate", "up") if gated else ("w",):
        s[p] = matrices(E, N, K)
        s["b_" + p] = normal((N,) if E is None else (E, N), 0.1, t) if case["bias"] else None
    s["residual"] = normal((M, N), 1.0, t) if case.get("residual") else None
    return s


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        from promoe_amd import ops
        for p in ("gate", "up", "w"):
            if p in state:
                state[p] = ops.Mx4(*state[p])
        if "idx" in state:
            state["dispatch"] = ops.dispatch(state["idx"], case["E"])
    if case.get("grad"):
        state["x"].requires_grad_(True)
        state["weights"].requires_grad_(True)
    return state


def _run_own(s):
    from promoe_amd import ops
    case, x = s["case"], s["x"]
    op, t = case["op"], TYPES[case["dtype"]]
    if op == "quantize":
        return ops.dequantize_mx4(ops.quantize_mx4(x), t)
    if op == "sort":
        y = ops.sort_tokens(x, s["dispatch"])
        return (y, *torch.autograd.grad(y, [x], s["g"])) if case["grad"] else y
    if op == "unsort":
        y = ops.unsort_tokens(x, s["dispatch"], s["weights"])
        return (y, *torch.autograd.grad(y, [x, s["weights"]], s["g"])) if case["grad"] else y
    out = torch.float32 if case.get("out") == "fp32" else t
    if case["x"] == "mx4":
        x = ops.quantize_mx4(x)
    if op == "experts":
        if case["gated"]:
            return ops.experts_gated_mx4(x, s["gate"], s["up"], s["dispatch"], s["b_gate"], s["b_up"], act=case["act"], of_tokens=True,
                                         out_dtype=t)
        return ops.experts_linear_mx4(x, s["w"], s["dispatch"], s["b_w"], out_dtype=t)
    if op == "linear":
        return ops.linear_mx4(x, s["w"], s["b_w"], act=case["act"], residual=s["residual"], out_dtype=out)
    return ops.linear_gated_mx4(x, s["gate"], s["up"], s["b_gate"], s["b_up"], act=case["act"], out_dtype=out)


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


def _by_expert(s, x, w, b):
    """Rows x (in the experts' order) times the matrix of their expert"""
    case = s["case"]
    E, P = case["E"], x.shape[0]
    which = torch.repeat_interleave(torch.arange(E, device=x.device), s["counts"], output_size=P)
    if P <= E:        # a matrix for each row
        y = torch.bmm(x[:, None], _unpacked((w[0][which], w[1][which])).transpose(1, 2).contiguous())[:, 0]
    else:             # experts of one size, the shorter ones with rows of zeros behind theirs
        first = torch.cumsum(s["counts"], 0) - s["counts"]
        place = torch.arange(P, device=x.device) - first[which]
        wide = torch.zeros(E, max(s["sizes"]), x.shape[1], device=x.device)
        wide[which, place] = x
        y = torch.bmm(wide, _unpacked(w).transpose(1, 2).contiguous())[which, place]
    return y if b is None else y + b.float()[which]


def run(s):
    if own:
        return _run_own(s)
    case, x = s["case"], s["x"].detach()
    op, t = case["op"], TYPES[case["dtype"]]
    if op == "quantize":
        return _rounded(x).to(t)
    if op in ("sort", "unsort"):
        T, k = case["T"], case["k"]
        here = (s["pos"] < s["here"])[:, None]
        if op == "sort":
            tok = s["order"] // k
            there = (torch.arange(T * k, device=x.device) < s["here"])[:, None]
            y = torch.where(there, x[tok], 0.0)
            if not case["grad"]:
                return y
            dx = torch.where(here, s["g"][s["pos"]].float(), 0.0).view(T, k, -1).sum(1)
            return y, dx.to(t)
        w = s["weights"].detach()
        rows = torch.where(here, x[s["pos"]].float(), 0.0).view(T, k, -1)
        y = (rows * w[:, :, None]).sum(1).to(t)
        if not case["grad"]:
            return y
        g = s["g"].float()[:, None]
        dw = (rows * g).sum(2)
        by_pair = torch.where(here, (w[:, :, None] * g).flatten(0, 1), 0.0)
        return y, by_pair[s["order"]].to(t), dw
    x = _rounded(x) if case["x"] == "mx4" else x.float()
    gated = case["gated"] if op == "experts" else op == "gated"
    if op == "experts":
        if gated:
            x = x[s["order"] // case["k"]]

        def product(p):
            return _by_expert(s, x, s[p], s["b_" + p])
    else:
        def product(p):
            v = x @ _unpacked(s[p]).t()
            return v if s["b_" + p] is None else v + s["b_" + p].float()

    y = _act(case["act"], product("gate")) * product("up") if gated else _act(case["act"], product("w"))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y if case.get("out") == "fp32" else y.to(t)


def _blocks64(x):
    """Quantised values in 64 bits, by counting the borders below a magnitude"""
    b = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = b.abs().max(dim=-1, keepdim=True).values
    e = torch.frexp(top).exponent.double() - 3.0          # floor(log2 top) - 2
    scale = torch.where(top > 0, torch.exp2(torch.clamp(e, min=-127.0)), torch.ones_like(top))
    r = b.abs() / scale
    n = torch.zeros_like(r, dtype=torch.int64)
    for border, even_below in ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)):
        n += (r > border) if even_below else (r >= border)
    v = torch.tensor(GRID, dtype=torch.float64, device=x.device)[n]
    return (torch.copysign(v, b) * scale).reshape(x.shape)


def _matrix64(codes, scales):
    """codes [N, K / 2], scales [N, K / 32] -> [N, K]: sign, two bits of exponent, one of mantissa"""
    c = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.int64, device=codes.device)
    c[:, 0::2] = codes & 15
    c[:, 1::2] = codes >> 4
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e > 0, (1.0 + m / 2) * torch.exp2(e.double() - 1), m / 2) * (1 - 2 * (c >> 3)).double()
    return v * torch.exp2(scales.double() - 127.0).repeat_interleave(32, dim=1)


def _product64(x, w, b):
    y = torch.empty(x.shape[0], w[0].shape[0], dtype=torch.float64, device=x.device)
    for j in range(0, y.shape[1], 1024):
        y[:, j: j + 1024] = torch.mm(x, _matrix64(w[0][j: j + 1024], w[1][j: j + 1024]).t().contiguous())
    return y if b is None else y + b.double()


def exact(case, seed):
    s = _inputs(case, seed)
    op, x = case["op"], s["x"]
    if op == "quantize":
        return _blocks64(x)
    if op in ("sort", "unsort"):
        T, k, H = case["T"], case["k"], case["H"]
        idx = s["idx"].reshape(-1)
        pairs = torch.cat([torch.nonzero(idx == e)[:, 0] for e in range(case["E"])])     # in the order of the experts
        n = pairs.numel()
        tok = pairs // k
        if op == "sort":
            y = torch.zeros(T * k, H, dtype=torch.float64, device=x.device)
            y[:n] = x.double()[tok]
            if not case["grad"]:
                return y
            return y, torch.zeros(T, H, dtype=torch.float64, device=x.device).index_add_(0, tok, s["g"].double()[:n])
        w = s["weights"].double().reshape(-1)
        rows = x.double()[:n]
        y = torch.zeros(T, H, dtype=torch.float64, device=x.device).index_add_(0, tok, rows * w[pairs, None])
        if not case["grad"]:
            return y
        g = s["g"].double()[tok]
        dx = torch.zeros(T * k, H, dtype=torch.float64, device=x.device)
        dx[:n] = g * w[pairs, None]
        dw = torch.zeros(T * k, dtype=torch.float64, device=x.device)
        dw[pairs] = (g * rows).sum(1)
        return y, dx, dw.view(T, k)
    fn = {"none": lambda v: v, "relu": lambda v: v * (v > 0), "relu2": lambda v: v * v * (v > 0),
          "silu": lambda v: v * torch.special.expit(v), "gelu": lambda v: v * (1 + torch.special.erf(v / math.sqrt(2))) / 2,
          "gelu_tanh": lambda v: v * (1 + torch.tanh((v + 0.044715 * v ** 3) * math.sqrt(2 / math.pi))) / 2}[case["act"]]
    x = _blocks64(x) if case["x"] == "mx4" else x.double()

    def layer(x, pick):
        """pick(p): matrix and bias of part p"""
        if (case["gated"] if op == "experts" else op == "gated"):
            return fn(_product64(x, *pick("gate"))) * _product64(x, *pick("up"))
        return fn(_product64(x, *pick("w")))

    if op != "experts":
        y = layer(x, lambda p: (s[p], s["b_" + p]))
        return y if s["residual"] is None else y + s["residual"].double()
    parts, at = [], 0
    tok = torch.sort(s["idx"].reshape(-1), stable=True).indices // case["k"]
    for e, n in enumerate(s["sizes"]):
        if n:
            rows = x[tok[at: at + n]] if case["gated"] else x[at: at + n]
            parts.append(layer(rows, lambda p: ((s[p][0][e], s[p][1][e]), None if s["b_" + p] is None else s["b_" + p][e])))
            at += n
    return torch.cat(parts)


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "fp32" else 2
    if op == "quantize":
        # read, 4.25 bits a value written and read, written; about eight operations a value
        M, K = case["M"], case["K"]
        return {"bytes": 2.0 * M * K * size + 2.0 * M * (K // 2 + K // 32), "flops": 8.0 * M * K}
    if op in ("sort", "unsort"):
        T, H, P = case["T"], case["H"], case["T"] * case["k"]
        # one way: the tokens' rows and the experts', places, weights
        nbytes, flops = size * H * (T + P) + 4.0 * P, 0.0 if op == "sort" else 2.0 * P * H
        if op == "unsort":
            nbytes += 4.0 * P
        if case["grad"]:
            # sort: the same rows the other way; unsort: gradients in, rows, gradients out, and of the weights
            nbytes += size * H * (T + P) + 4.0 * P if op == "sort" else size * H * (T + 2 * P) + 12.0 * P
            flops += P * H if op == "sort" else 3.0 * P * H
        return {"bytes": nbytes, "flops": flops}
    N, K = case["N"], case["K"]
    gated = case["gated"] if op == "experts" else op == "gated"
    mats = 2 if gated else 1
    if op == "experts":
        T, E, k = case["T"], case["E"], case["k"]
        M, rows_in, used = T * k, T if gated else T * k, E * (1.0 - (1.0 - k / E) ** T)
    else:
        M, rows_in, used = case["M"], case["M"], 1.0
    nbytes = rows_in * K * 2.0 + used * mats * N * (K // 2 + K // 32) + M * N * (4.0 if case.get("out") == "fp32" else 2.0)
    nbytes += 2.0 * used * mats * N if case["bias"] else 0.0
    nbytes += 2.0 * M * N if case.get("residual") else 0.0
    return {"bytes": nbytes, "flops": 2.0 * mats * M * N * K}
