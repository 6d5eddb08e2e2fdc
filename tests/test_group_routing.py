"""Routing with groups and a selection bias: the oracle against brute force, and what the entry points refuse (no GPU needed)."""
import ctypes
import itertools

import numpy as np
import pytest
import torch

from oracle import moe_oracle as O
from oracle import route_oracle as R


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_value", ["max", "top2"])
def test_oracle_is_the_best_subset(kind, group_value):
    """Among all choices of topk_group groups and then of k experts inside them, the one whose values add up to most."""
    rng = np.random.default_rng(3)
    lg = rng.normal(0, 1.5, (40, 8)).astype(np.float32)
    bias = rng.normal(0, 0.2, 8).astype(np.float32)
    idx, w = R.route(lg, 3, kind, bias, 4, 2, group_value)
    s = R.scores(lg, kind)
    c = s + bias.astype(np.float64)
    for t in range(40):
        worth = [(c[t, 2 * g: 2 * g + 2].sum() if group_value == "top2" else c[t, 2 * g: 2 * g + 2].max()) for g in range(4)]
        kept = max(itertools.combinations(range(4), 2), key=lambda gs: sum(worth[g] for g in gs))
        cand = [e for g in kept for e in (2 * g, 2 * g + 1)]
        best = max(itertools.combinations(cand, 3), key=lambda es: sum(c[t, e] for e in es))
        assert set(idx[t]) == set(best)
        assert np.all(np.diff(c[t, idx[t]]) <= 0) and np.array_equal(w[t], s[t, idx[t]])


def test_oracle_without_groups_is_the_plain_router():
    lg = np.random.default_rng(5).normal(0, 1.5, (50, 24)).astype(np.float32)
    for renorm, mode in ((False, 0), (True, 1)):
        idx, w = R.route(lg, 5, renorm=renorm)
        ridx, rw = O.topk_route(lg, 5, mode)
        assert np.array_equal(idx, ridx) and np.allclose(w, rw, rtol=1e-5, atol=0)


def test_refusals_at_the_c_entries():
    from promoe_amd import _lib as L
    p = 4096                                     # never read

    def rule(**kw):
        d = dict(scores=0, n_group=4, topk_group=2, group_value=0, renorm=0, scale=1.0)
        d.update(kw)
        return L.RouteRule(**d)

    def topk(r, T=2, E=16, ldl=16, k=4, logits=p):
        return L.lib.moe_group_topk(logits, T, E, ldl, k, None if r is None else ctypes.byref(r), p, p, p, None)

    def disp(r, T=2, E=16, k=4):
        return L.lib.moe_group_topk_dispatch(p, T, E, E, k, ctypes.byref(r), p, *([p] * 10), min(E, T * k), None, None, None, 0, None)

    bad = [dict(scores=2), dict(scores=-1), dict(n_group=0), dict(n_group=3), dict(topk_group=0), dict(topk_group=5),
           dict(group_value=2), dict(topk_group=1, n_group=8), dict(n_group=16, topk_group=8, group_value=1)]
    for kw in bad:
        assert topk(rule(**kw)) == L.MOE_EINVAL and b"rule" in L.lib.moe_last_error(), kw
        assert disp(rule(**kw)) == L.MOE_EINVAL, kw
    assert topk(None) == L.MOE_EINVAL
    for kw in (dict(T=-1), dict(ldl=15), dict(k=0), dict(k=33, E=256, ldl=256), dict(E=260, ldl=260), dict(logits=None)):
        assert topk(rule(), **kw) == L.MOE_EINVAL, kw
    for kw in (dict(T=0), dict(T=65, k=1), dict(T=64, k=9, E=64)):
        assert disp(rule(n_group=2, topk_group=2), **kw) == L.MOE_EINVAL, kw
    assert topk(rule(), T=0, logits=None) == 0   # nothing to do


def test_refusals_of_the_wrappers():
    from promoe_amd import _lib as L
    from promoe_amd import ops
    with pytest.raises(L.MoeError, match="scores"):
        ops.RouteRule("tanh")
    with pytest.raises(L.MoeError, match="group_value"):
        ops.RouteRule(group_value="mean")
    r = ops.RouteRule("sigmoid", 2, 1, "top2")
    for lg in (torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(8), torch.zeros(3, 16)[:, ::2]):
        with pytest.raises(L.MoeError):
            ops.group_topk(lg, 2, r)
        with pytest.raises(L.MoeError):
            ops.group_topk_dispatch(lg, 2, r)
    with pytest.raises(L.MoeError, match="rule"):
        ops.group_topk(torch.zeros(3, 8), 2, None)


def test_an_engine_refuses_a_rule_for_a_layer_it_does_not_know():
    from promoe_amd import _lib as L
    from promoe_amd.engine import ModuleMeta, PrefetchMngr
    m = ModuleMeta(2, 8)
    m.init_param_list(["w"])
    m.init_from_map({"num_expert_per_token": "2"})
    m.handle_uninited_configs()
    pm = PrefetchMngr(m, backend=L.BACKEND_HOST)
    r = L.RouteRule(1, 2, 1, 1, 1, 1.0)
    assert L.lib.moe_set_layer_routing(pm._h, 2, ctypes.byref(r), None) == L.MOE_EINVAL
    assert L.lib.moe_set_layer_routing(pm._h, 0, ctypes.byref(r), None) == L.MOE_ESTATE
    assert L.lib.moe_set_layer_routing(None, 0, ctypes.byref(r), None) == L.MOE_EINVAL
    d = L.LayerDesc(128, 128, 0, 5, 0, L.FMT_INT4_G128, 0, 4096, None, None)
    L.check(L.lib.moe_set_layer(pm._h, 0, ctypes.byref(d)))
    assert L.lib.moe_set_layer_routing(pm._h, 0, ctypes.byref(r), None) == L.MOE_EINVAL       # 5 choices, 4 experts in a group
    r.topk_group = 2
    assert L.lib.moe_set_layer_routing(pm._h, 0, ctypes.byref(r), None) == 0
    assert L.lib.moe_set_layer_routing(pm._h, 0, None, None) == 0
    pm.close()
