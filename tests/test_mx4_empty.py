"""Matrices in 4 bits of no rows, or none of them (no GPU needed: nothing is launched)."""
import pytest
import torch


@pytest.mark.parametrize("shape", [(0, 64), (0, 5, 64), (3, 0, 64), (0, 0, 32), (1, 0, 96)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nothing_is_quantised_to_nothing(monkeypatch, shape, dtype):
    from promoe_amd import ops
    monkeypatch.setattr(ops, "_operands", lambda what, first, *others: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    q = ops.quantize_mx4(torch.empty(shape, dtype=dtype))
    assert q.shape == shape and q.codes.shape == (*shape[:-1], shape[-1] // 2) and q.scales.shape == (*shape[:-1], shape[-1] // 32)
    y = ops.dequantize_mx4(q, dtype)
    assert y.shape == shape and y.dtype == dtype
    assert ops.Mx4(q.codes, q.scales).shape == shape


@pytest.mark.gpu
def test_nothing_on_the_gpu(cuda):
    from promoe_amd import ops
    print("case mx4_empty", flush=True)
    for shape in ((0, 64), (0, 5, 64), (3, 0, 64)):
        x = torch.empty(shape, dtype=torch.bfloat16, device=cuda)
        assert ops.dequantize_mx4(ops.quantize_mx4(x)).shape == shape
    E, T, k = 8, 0, 2                                          # and no tokens for any expert
    d = ops.dispatch(torch.empty(T, k, dtype=torch.int32, device=cuda), E)
    w = ops.quantize_mx4(torch.randn(E, 96, 64, device=cuda))
    x = torch.empty(T, 64, dtype=torch.bfloat16, device=cuda)
    for q in (lambda t: t, ops.quantize_mx4):
        h = ops.experts_gated_mx4(q(x), w, w, d, of_tokens=True)
        assert h.shape == (0, 96)
    assert ops.sort_tokens(x, d).shape == (0, 64) and ops.unsort_tokens(x, d, torch.empty(T, k, device=cuda)).shape == (0, 64)
