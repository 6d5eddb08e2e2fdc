"""CPU restatement of routing with groups of experts and a selection bias, in 64 bits (TEST INFRASTRUCTURE ONLY).

Pinned by the closed form itself, by brute force over all subsets on tiny inputs (tests/test_group_routing.py), by the router
without groups (oracle/moe_oracle.py) where the rule has none, and by a stock transformers model with a group-limited router run
through the engine (tests/test_hf_dense_gpu.py)."""
from __future__ import annotations

import numpy as np


def scores(logits: np.ndarray, kind: str) -> np.ndarray:
    l = np.asarray(logits, np.float32).astype(np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    with np.errstate(all="ignore"):
        if kind == "sigmoid":
            return 1.0 / (1.0 + np.exp(-l))
        m = l.max(axis=1, keepdims=True)
        e = np.exp(l - m)
        s = e / e.sum(axis=1, keepdims=True)
    s[np.isneginf(m[:, 0])] = 0.0
    return s


def route(logits, k, kind="softmax", bias=None, n_group=1, topk_group=1, group_value="max", renorm=False, scale=1.0):
    """(idx [T, k] int32, w [T, k] float64)"""
    s = scores(logits, kind)
    T, E = s.shape
    c = s if bias is None else s + np.asarray(bias, np.float64)
    c = np.where(np.isnan(c), -np.inf, c)
    size = E // n_group
    idx = np.empty((T, k), np.int32)
    w = np.empty((T, k))
    for t in range(T):
        groups = [sorted(c[t, g * size: (g + 1) * size], reverse=True) for g in range(n_group)]
        with np.errstate(all="ignore"):
            v = [g[0] + g[1] if group_value == "top2" and size > 1 else g[0] for g in groups]
        v = [-np.inf if np.isnan(x) else x for x in v]
        kept = sorted(range(n_group), key=lambda g: (-v[g], g))[:topk_group]
        cand = [e for g in kept for e in range(g * size, (g + 1) * size)]
        idx[t] = sorted(cand, key=lambda e: (-c[t, e], e))[:k]
        w[t] = s[t, idx[t]]
        if renorm:
            total = w[t].sum()
            w[t] = w[t] / total if total != 0.0 else 0.0
        w[t] *= scale
    return idx, w
