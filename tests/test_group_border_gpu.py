"""Which groups stay where their values are hard to tell apart: group_topk and its dispatch against the definition in 64 bits (whole
numbers equal, weights off by their one rounding to fp32)."""
import numpy as np
import pytest
import torch

from oracle import route_oracle as R

pytestmark = pytest.mark.gpu


def _many(lg, k, kind, bias, G, keep, renorm=False):
    """The oracle's route for groups worth their two largest, all rows at once: (idx, w)."""
    s = R.scores(lg, kind)
    T, E = s.shape
    c = s + bias.astype(np.float64)
    g = np.sort(c.reshape(T, G, E // G), axis=2)
    order = np.argsort(-(g[:, :, -1] + g[:, :, -2]), axis=1, kind="stable")[:, :keep]
    kept = np.zeros((T, G), bool)
    np.put_along_axis(kept, order, True, axis=1)
    idx = np.argsort(-np.where(np.repeat(kept, E // G, axis=1), c, -np.inf), axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(s, idx, axis=1)
    return idx.astype(np.int32), w / w.sum(axis=1, keepdims=True) if renorm else w


def _check(lg, k, kind, bias, G, keep, dev):
    from promoe_amd import ops
    rule = ops.RouteRule(kind, G, keep, "top2")
    ld, bd = torch.from_numpy(lg).to(dev), torch.from_numpy(bias).to(dev)
    ridx, rw = _many(lg, k, kind, bias, G, keep)
    for a, b in zip(_many(lg[:6], k, kind, bias, G, keep), R.route(lg[:6], k, kind, bias, G, keep, "top2")):
        assert np.array_equal(a, b)
    n = min(len(lg), 64, 512 // k)
    for idx, w in (ops.group_topk(ld, k, rule, bd), ops.group_topk_dispatch(ld[:n], k, rule, bd)[:2]):
        idx, w = idx.cpu().numpy(), w.cpu().numpy().astype(np.float64)
        bad = (idx != ridx[: len(idx)]).any(axis=1)
        assert not bad.any(), "%d of %d rows" % (bad.sum(), len(idx))
        assert (np.abs(w - rw[: len(w)]) <= 2.0 ** -24 * 1.001 * rw[: len(w)] + 2.0 ** -149).all()


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,k,G,keep", [(16, 1, 8, 1), (16, 2, 8, 4), (24, 3, 3, 1), (60, 4, 6, 3), (256, 8, 8, 4), (32, 4, 16, 5),
                                        (128, 2, 64, 7)])
def test_groups_of_equal_value(cuda, E, k, G, keep, kind):
    """Sums that are equal although what they are made of is not (3 + 2, 4 + 1), at the border between the groups that stay and the
    others: the lower group stays, and one expert more or less would be chosen with the other."""
    print(f"case group_equal {E} {k} {G} {keep} {kind}", flush=True)
    for seed in range(24):
        rng = np.random.default_rng(seed)
        bias = (rng.integers(-8, 9, E) * 0.5).astype(np.float32)
        # (scores of zero, one half and one; softmax: all the same, or one expert's alone)
        lg = rng.choice(np.array([0.0, 200.0, -200.0], np.float32), (65, E))
        if kind == "softmax":
            lg[::2] = 0.0
        _check(lg, k, kind, bias, G, keep, cuda)


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size", [2, 4, 32])
def test_biases_of_both_signs(cuda, size, kind):
    """A group's two largest are one of a large positive and one of a large negative bias (the others are behind both), so that
    its value is what 32 bits have lost of them."""
    T, G, keep = 65536, 8, 4
    for big in (1.0, 16.0, 64.0, 256.0, 1e3, 1e4, 1e5, 1e6):
        print(f"case group_cancel size={size} {kind} bias={big}", flush=True)
        rng = np.random.default_rng(size)
        lg = rng.normal(0, 1.2, (T, G * size)).astype(np.float32)
        sign = np.full((G, size), -3.0)
        sign[:, :2] = (1.0, -1.0)
        bias = (sign * big + rng.normal(0, 0.05, (G, size))).astype(np.float32).reshape(-1)
        _check(lg, 4, kind, bias, G, keep, cuda)


def test_infinite_biases(cuda):
    """-inf takes an expert out of the choice (of its group's value too), one +inf puts a group in front, two of them are equal
    groups: the lower one."""
    print("case group_infinite", flush=True)
    rng = np.random.default_rng(4)
    lg = rng.normal(0, 1.2, (300, 64)).astype(np.float32)
    for at, v in (((3, 17, 40), -np.inf), ((9,), np.inf), ((9, 33), np.inf), ((9, 33, 50), np.inf)):
        bias = rng.normal(0, 0.05, 64).astype(np.float32)
        bias[list(at)] = v
        for keep in (1, 2, 5):
            _check(lg, 4, "sigmoid", bias, 8, keep, cuda)


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
def test_scores_at_the_end_of_the_range(cuda, kind):
    """The bias chooses experts whose scores are the smallest that 64 bits hold, or nothing: renormalised, they are what counts.  The
    form for few tokens a wave (rows 2^26 + 4 floats apart take it throughout) has the same bits; sigmoids past e^709 are zero, and so
    are weights of nothing else."""
    from promoe_amd import ops
    print(f"case group_tiny {kind}", flush=True)
    E, k, T, ldl = 64, 4, 24, (1 << 26) + 4
    rng = np.random.default_rng(6)
    lg = rng.uniform(-760, -690, (T, E)).astype(np.float32)
    lg[:4] = rng.uniform(-745, -711, (4, E)).astype(np.float32)
    if kind == "softmax":
        lg[:, 0] = 0.0
    bias = np.full(E, -8.0, np.float32)
    bias[[5, 17, 30, 41]] = (4.0, 2.0, 8.0, 6.0)                     # far apart: 32 bits are certain of these
    far = torch.empty((T - 1) * ldl + E, device=cuda).as_strided((T, E), (ldl, 1))
    far.copy_(torch.from_numpy(lg))
    bd = torch.from_numpy(bias).to(cuda)
    for G, keep, gv in ((1, 1, "max"), (8, 4, "max")):
        rule = ops.RouteRule(kind, G, keep, gv, True, 1.0)
        idx, w = ops.group_topk(far.contiguous(), k, rule, bd)
        i2, w2 = ops.group_topk(far, k, rule, bd)
        assert (idx.cpu() == torch.tensor([30, 41, 5, 17], dtype=torch.int32)).all() and torch.equal(idx, i2)
        assert torch.equal(w, w2), int((w != w2).any(1).sum())
        i3, w3, _ = ops.group_topk_dispatch(far.contiguous(), k, rule, bd)
        assert torch.equal(idx, i3) and torch.equal(w, w3)
        if kind == "sigmoid":
            assert (w[:4] == 0).all()
            ref = R.route(lg, k, kind, bias, G, keep, gv, True, 1.0)[1]
            assert np.array_equal(w.cpu().numpy() == 0, ref.astype(np.float32) == 0)
