"""Routing with groups and a selection bias on the GPU, against the oracle in 64 bits: whole numbers equal, weights off by their
one rounding to fp32 (2^-24 of the value; the 64-bit arithmetic on both sides adds under 2^-40)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import moe_oracle as O
from oracle import route_oracle as R
from tests.synth import Bf16Layer, Int4Layer, Q4KLayer

pytestmark = pytest.mark.gpu

RULES = [  # E, k, scores, bias, n_group, topk_group, group_value, renorm, scale
    (64, 6, "sigmoid", True, 1, 1, "max", True, 1.0),
    (64, 6, "softmax", False, 8, 3, "max", False, 16.0),
    (60, 4, "softmax", True, 6, 3, "top2", True, 1.0),
    (8, 2, "sigmoid", False, 1, 1, "max", False, 1.0),
    (1, 1, "softmax", False, 1, 1, "max", True, 1.0),
    (256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5),
    (250, 32, "softmax", True, 5, 4, "max", False, 1.0),
    (128, 8, "sigmoid", True, 64, 32, "top2", False, 1.0),
    (63, 7, "sigmoid", True, 63, 9, "max", True, 1.0),
    (160, 6, "softmax", False, 8, 3, "max", False, 16.0),
    (192, 5, "sigmoid", True, 3, 3, "max", True, 1.0),
]


def _rule(c):
    from promoe_amd import ops
    return ops.RouteRule(c[2], c[4], c[5], c[6], c[7], c[8])


def _ref(lg, c, bias):
    return R.route(lg, c[1], c[2], bias, *c[4:])


def _data(c, T, seed, dev, spread=1.5, gap=0):
    rng = np.random.default_rng(seed)
    lg = rng.normal(0, spread, (T, c[0])).astype(np.float32)
    bias = rng.normal(0, 0.05, c[0]).astype(np.float32) if c[3] else None
    wide = np.full((T, c[0] + gap), np.nan, np.float32)
    wide[:, :c[0]] = lg
    return lg, bias, torch.from_numpy(wide).to(dev)[:, :c[0]], None if bias is None else torch.from_numpy(bias).to(dev)


def _close(w, ref):
    assert np.all(np.abs(w.astype(np.float64) - ref) <= 2.0 ** -24 * 1.001 * np.abs(ref) + 2.0 ** -149), np.abs(w - ref).max()


@pytest.mark.parametrize("T,gap", [(1, 0), (3, 1), (4, 0), (65, 3), (1023, 1)])
@pytest.mark.parametrize("c", RULES, ids=lambda c: "-".join(str(v) for v in c[:7]))
def test_group_topk(cuda, c, T, gap):
    from promoe_amd import ops
    print(f"case group_topk {c} T={T} gap={gap}", flush=True)
    lg, bias, ld, bd = _data(c, T, 11 * T + c[0], cuda, gap=gap)
    idx, w = ops.group_topk(ld, c[1], _rule(c), bd)
    ridx, rw = _ref(lg, c, bias)
    assert np.array_equal(idx.cpu().numpy(), ridx)
    _close(w.cpu().numpy(), rw)


@pytest.mark.parametrize("T", [1, 2, 4, 5, 16, 33, 64])
@pytest.mark.parametrize("c", RULES, ids=lambda c: "-".join(str(v) for v in c[:7]))
def test_group_topk_dispatch(cuda, c, T):
    from promoe_amd import ops
    T = min(T, 512 // c[1])
    print(f"case group_topk_dispatch {c} T={T}", flush=True)
    lg, bias, ld, bd = _data(c, T, 13 * T + c[0], cuda, gap=1)
    idx, w, d = ops.group_topk_dispatch(ld, c[1], _rule(c), bd)
    ridx, rw = _ref(lg, c, bias)
    assert np.array_equal(idx.cpu().numpy(), ridx)
    _close(w.cpu().numpy(), rw)
    ref = ops.dispatch(torch.from_numpy(ridx).to(cuda), c[0], single_workgroup=True)
    for n in ("counts", "offsets", "sorted_pair", "pos_of_pair", "sorted_tok", "units", "n_active", "active_ids"):
        assert torch.equal(getattr(d, n), getattr(ref, n)), n


@pytest.mark.parametrize("c", [r for r in RULES if r[0] in (64, 60, 256, 63)], ids=lambda c: "-".join(str(v) for v in c[:7]))
def test_ties_and_close_values(cuda, c):
    """Logits of a few values (equal scores everywhere: the lower expert, the lower group), and logits a rounding of 32 bits apart
    (saturated sigmoids and scores whose fp32 values are equal: the larger 64-bit score)."""
    from promoe_amd import ops
    E, T = c[0], 200
    print(f"case group_topk_ties {c}", flush=True)
    rng = np.random.default_rng(E)
    few = rng.integers(-2, 3, (T, E)).astype(np.float32)
    close = (np.float32(0.75) * (1 + rng.integers(-3, 4, (T, E)) * np.float32(2.0) ** -22)).astype(np.float32)
    large = (14 + rng.integers(0, 8, (T, E)) * 0.25).astype(np.float32)
    for lg in (few, close, large):
        bias = (rng.integers(-2, 3, E) * np.float32(2.0) ** -26).astype(np.float32) if c[3] else None
        idx, w = ops.group_topk(torch.from_numpy(lg).to(cuda), c[1], _rule(c), None if bias is None else torch.from_numpy(bias).to(cuda))
        ridx, rw = _ref(lg, c, bias)
        assert np.array_equal(idx.cpu().numpy(), ridx)
        _close(w.cpu().numpy(), rw)


@pytest.mark.parametrize("c", RULES, ids=lambda c: "-".join(str(v) for v in c[:7]))
def test_masked_rows_infinities_and_nan(cuda, c):
    """Rows with -inf, the type's lowest value, NaN, and with nothing else; k different experts whatever the row."""
    from promoe_amd import ops
    E, k = c[0], c[1]
    print(f"case group_topk_masks {c}", flush=True)
    lg, bias, _, bd = _data(c, 12, 7 + E, cuda)
    low = np.finfo(np.float32).min
    lg[0] = -np.inf
    lg[1] = np.nan
    lg[2] = low
    lg[3, : E // 2] = -np.inf
    lg[4, E // 2:] = np.nan
    lg[5, 1:] = low
    lg[6, : E - 1] = -np.inf
    lg[7] = 80.0
    lg[8] = -120.0
    lg[9, ::3] = -np.inf
    ld = torch.from_numpy(lg).to(cuda)
    idx, w = ops.group_topk(ld, k, _rule(c), bd)
    ridx, rw = _ref(lg, c, bias)
    assert np.array_equal(idx.cpu().numpy(), ridx)
    _close(w.cpu().numpy(), rw)
    if c[2] == "softmax":
        assert np.all(w.cpu().numpy()[:2] == 0.0)
    # +inf, and a bias of NaN: still k different experts
    lg[:, 0] = np.inf
    lg[3] = np.inf
    bad = None if bd is None else torch.where(torch.arange(E, device=cuda) % 5 == 1, float("nan"), bd)
    idx = ops.group_topk(torch.from_numpy(lg).to(cuda), k, _rule(c), bad)[0].cpu().numpy()
    assert all(len(set(r)) == k and min(r) >= 0 and max(r) < E for r in idx)
    i2 = ops.group_topk_dispatch(torch.from_numpy(lg).to(cuda), k, _rule(c), bad)[0].cpu().numpy()
    assert np.array_equal(idx, i2)


def test_empty_batch_other_stream_and_graph(cuda):
    from promoe_amd import ops
    print("case group_topk_graph", flush=True)
    c = RULES[5]
    idx, w = ops.group_topk(torch.empty(0, c[0], device=cuda), c[1], _rule(c))
    assert idx.shape == (0, c[1]) and w.shape == (0, c[1])
    lg, bias, ld, bd = _data(c, 33, 5, cuda)
    ld = ld.contiguous()
    rule = _rule(c)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a = ops.group_topk(ld, c[1], rule, bd)
    torch.cuda.synchronize()
    ridx, rw = _ref(lg, c, bias)
    assert np.array_equal(a[0].cpu().numpy(), ridx)
    x = ld.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b = ops.group_topk(x, c[1], rule, bd)
        idx, w, d = ops.group_topk_dispatch(x, c[1], rule, bd)
    for seed in range(4):
        lg, _, nd, _ = _data(c, 33, 100 + seed, cuda)
        x.copy_(nd)
        g.replay()
        torch.cuda.synchronize()
        ridx, rw = _ref(lg, c, bias)
        assert np.array_equal(b[0].cpu().numpy(), ridx) and np.array_equal(idx.cpu().numpy(), ridx)
        _close(b[1].cpu().numpy(), rw)
        ref = ops.dispatch(torch.from_numpy(ridx).to(cuda), c[0], single_workgroup=True)
        assert torch.equal(d.sorted_pair, ref.sorted_pair) and torch.equal(d.units, ref.units)


def test_gradients_are_refused(cuda):
    from promoe_amd import _lib as L
    from promoe_amd import ops
    x = torch.zeros(2, 8, device=cuda, requires_grad=True)
    with pytest.raises(L.MoeError, match="gradient"):
        ops.group_topk(x, 2, ops.RouteRule())
    with torch.no_grad():
        assert ops.group_topk(x, 2, ops.RouteRule())[0].tolist() == [[0, 1], [0, 1]]


@pytest.mark.parametrize("cache_rate", [1.0, 0.5])
@pytest.mark.parametrize("kind", ["int4", "bf16", "q4k"])
def test_layer_forward_with_groups(cuda, kind, cache_rate):
    """moe_forward of a layer with such a router, every batch path, against the oracle's routing and experts; and the same layer by
    its route mode again afterwards."""
    from promoe_amd import _lib as L
    from tests.test_engine_gpu import build_engine, ref_forward
    mk = {"int4": Int4Layer, "bf16": Bf16Layer, "q4k": Q4KLayer}[kind]
    E, k = 16, 4
    layers = [mk(H=256, I=256, E=E, I_sh=256, seed=70 + i) for i in range(2)]
    rules = [(E, k, "sigmoid", True, 4, 2, "top2", True, 2.5), (E, k, "softmax", False, 8, 3, "max", False, 1.0)]
    bias = np.random.default_rng(1).normal(0, 0.1, E).astype(np.float32)
    bd = torch.from_numpy(bias).to(cuda)
    pm = build_engine(layers, k, cuda, max_tokens=700, cache_rate=cache_rate, cache_policy="lru")
    for l, c in enumerate(rules):
        L.check(L.lib.moe_set_layer_routing(pm._h, l, ctypes.byref(_rule(c)), L.ptr(bd) if c[3] else 0))
    if cache_rate == 1.0:
        for l in range(2):
            pm.acquire_layer(l, np.arange(E, dtype=np.int64))
            pm.release_layer(l)
        pm.drain()
    for T in (1, 1, 2, 8, 12, 17, 32, 33, 65, 300, 700):
        print(f"case group_layer kind={kind} cache={cache_rate} T={T}", flush=True)
        for l, (layer, c) in enumerate(zip(layers, rules)):
            x = O.synth_acts(T, 256, seed=T + l)
            y = pm.forward(l, torch.from_numpy(x).to(torch.bfloat16).to(cuda)).float().cpu().numpy()
            torch.cuda.synchronize()
            lg = O.gate_logits_ordered(x, layer.wg)
            idx, w = _ref(lg, c, bias if c[3] else None)
            assert np.array_equal(pm.last_routing_idx(T, k), idx)
            xt = torch.from_numpy(x)
            ref = O.swiglu_expert(xt, *[torch.from_numpy(np.asarray(a, np.float32)) for a in layer.shared_fp32])
            for e in range(E):
                tok, slot = np.nonzero(idx == e)
                if len(tok):
                    ws = [torch.from_numpy(np.asarray(a, np.float32)) for a in layer.experts_fp32[e]]
                    ref.index_add_(0, torch.from_numpy(tok), O.swiglu_expert(xt[tok], *ws) * torch.from_numpy(w[tok, slot]).float()[:, None])
            ref = ref.numpy()
            err = np.abs(y - ref).max() / np.abs(ref).max()
            assert err <= 2e-2, (T, l, err)
    L.check(L.lib.moe_set_layer_routing(pm._h, 0, None, None))
    x = O.synth_acts(4, 256, seed=9)
    y = pm.forward(0, torch.from_numpy(x).to(torch.bfloat16).to(cuda)).float().cpu().numpy()
    ref = ref_forward(layers[0], x, k, 0)["out"]
    assert np.abs(y - ref).max() / np.abs(ref).max() <= 2e-2
    pm.drain()
    pm.close()


@pytest.mark.parametrize("ldl", [1 << 26, (1 << 26) + 4])
def test_rows_far_apart(cuda, ldl):
    """Rows at both sides of the distance that four of them may have, far enough for offsets past 2^31: as rows side by side."""
    from promoe_amd import ops
    print(f"case group_topk_far ldl={ldl}", flush=True)
    c = RULES[5]
    _, _, ld, bd = _data(c, 37, 3, cuda)
    far = torch.empty(36 * ldl + c[0], device=cuda).as_strided((37, c[0]), (ldl, 1))
    far.copy_(ld)
    for f in (ops.group_topk, ops.group_topk_dispatch):
        a, b = f(ld, c[1], _rule(c), bd), f(far, c[1], _rule(c), bd)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_logits_and_bias_on_any_float(cuda):
    """Views that start at any float, in the middle of larger buffers, and end with them."""
    from promoe_amd import ops
    print("case group_topk_any_float", flush=True)
    for c in (RULES[5], RULES[2], RULES[0]):
        lg, bias, _, _ = _data(c, 13, 21, cuda)
        ridx, rw = _ref(lg, c, bias)
        for off in range(4):
            for gap in (0, 1, 2, 5):
                row = c[0] + gap
                buf = torch.full((off + 12 * row + c[0],), float("nan"), device=cuda)
                v = buf[off:].as_strided((13, c[0]), (row, 1), off)
                v.copy_(torch.from_numpy(lg))
                b = torch.full((off + c[0],), float("nan"), device=cuda)[off:]
                b.copy_(torch.from_numpy(bias))
                idx, w = ops.group_topk(v, c[1], _rule(c), b)
                assert np.array_equal(idx.cpu().numpy(), ridx)
                _close(w.cpu().numpy(), rw)
