"""Operators that have no forward-mode gradient refuse tensors with a tangent (no GPU needed: before anything else is looked at)."""
import pytest
import torch
from torch.autograd import forward_ad


def calls(dual):
    """Every wrapper with `dual` in the place of each operand that could have a tangent"""
    from promoe_amd import ops
    u8 = dict(dtype=torch.uint8)
    d = ops.Dispatch(4, 2, 3, 3, "cpu")
    q, qe = ops.Mx4(torch.zeros(8, 32, **u8), torch.zeros(8, 2, **u8)), ops.Mx4(torch.zeros(3, 8, 32, **u8), torch.zeros(3, 8, 2, **u8))
    bf = dict(dtype=torch.bfloat16)
    x, w, b, r = torch.zeros(4, 64, **bf), torch.zeros(8, 64, **bf), torch.zeros(8, **bf), torch.zeros(4, 8, **bf)
    rows, weights, logits = torch.zeros(8, 64, **bf), torch.zeros(4, 2), torch.zeros(4, 3)
    return {
        "sort x": lambda: ops.sort_tokens(dual(x), d), "unsort x": lambda: ops.unsort_tokens(dual(rows), d, weights),
        "unsort w": lambda: ops.unsort_tokens(rows, d, dual(weights)), "unsort x alone": lambda: ops.unsort_tokens(dual(rows), d),
        "quantize": lambda: ops.quantize_mx4(dual(x)), "linear_mx4 x": lambda: ops.linear_mx4(dual(x), q),
        "linear_mx4 bias": lambda: ops.linear_mx4(x, q, dual(b)), "linear_mx4 residual": lambda: ops.linear_mx4(x, q, residual=dual(r)),
        "linear_gated_mx4 b_up": lambda: ops.linear_gated_mx4(x, q, q, b, dual(b)), "experts x": lambda: ops.experts_linear_mx4(dual(rows), qe, d),
        "experts_gated bias": lambda: ops.experts_gated_mx4(x, qe, qe, d, b_up=dual(torch.zeros(3, 8, **bf)), of_tokens=True),
        "linear x": lambda: ops.linear(dual(x), w), "linear w": lambda: ops.linear(x, dual(w)), "linear residual": lambda: ops.linear(x, w, residual=dual(r)),
        "linear_gated b": lambda: ops.linear_gated(x, w, w, dual(b)), "group_topk": lambda: ops.group_topk(dual(logits), 2, ops.RouteRule()),
        "group_topk bias": lambda: ops.group_topk(logits, 2, ops.RouteRule(), dual(torch.zeros(3))),
    }


@pytest.mark.parametrize("name", sorted(calls(lambda t: t)))
def test_tensors_with_a_tangent_are_refused(name):
    from promoe_amd import _lib as L
    with forward_ad.dual_level():
        with pytest.raises(L.MoeError, match="forward-mode"):
            calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))[name]()


def test_tensors_without_one_are_not():
    """Past that check (these tensors of the CPU are refused for another reason): inside of a level without a tangent, the primal of a
    dual tensor, where forward mode is off (the forward pass of a function with a jvp of its own), and behind detach()."""
    from promoe_amd import _lib as L

    def passes(dual):
        for name, call in calls(dual).items():
            with pytest.raises(L.MoeError) as e:
                call()
            assert "forward-mode" not in str(e.value), name

    passes(lambda t: t)
    with forward_ad.dual_level():
        passes(lambda t: t)
        make = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        passes(lambda t: forward_ad.unpack_dual(make(t)).primal)
        passes(lambda t: make(t).detach())

        class Own(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x):
                passes(lambda t: x if t.shape == x.shape and t.dtype == x.dtype else t)
                return x * 2

            @staticmethod
            def jvp(ctx, g):
                return g * 2

        assert forward_ad.unpack_dual(Own.apply(make(torch.zeros(4, 64, dtype=torch.bfloat16)))).tangent is not None
