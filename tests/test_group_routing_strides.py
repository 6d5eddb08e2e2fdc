"""Rows of logits further apart than the entry points' 32-bit distance are refused, not read at what is left of it (no GPU needed)."""
import pytest
import torch


@pytest.mark.parametrize("apart", [1 << 31, (1 << 32) + 16, (1 << 33) + 20])
@pytest.mark.parametrize("fn", ["group_topk", "group_topk_dispatch"])
def test_rows_too_far_apart(fn, apart):
    from promoe_amd import _lib as L
    from promoe_amd import ops
    rule = ops.RouteRule("sigmoid", 2, 1, "top2")
    with pytest.raises(L.MoeError, match="apart"):
        getattr(ops, fn)(torch.empty_strided((3, 16), (apart, 1), device="meta"), 2, rule)
    # (one row has no distance; the next complaint is that it is not on a GPU)
    for t in (torch.empty_strided((1, 16), (apart, 1), device="meta"), torch.empty_strided((3, 16), ((1 << 31) - 1, 1), device="meta")):
        with pytest.raises(L.MoeError, match="GPU"):
            getattr(ops, fn)(t, 2, rule)
