"""gelu in fp32 results, against the formula in 64 bits.  One column of x times one: the sum is the value itself."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _exact(v):
    """(gelu, the half of erfc(|v| / sqrt 2) that it is made of)"""
    from scipy.special import erfc
    h = erfc(np.abs(v) / np.sqrt(2.0)) / 2
    return v * np.where(v > 0, 1 - h, h), h


@pytest.mark.parametrize("M", [1, 16, 300])                       # few rows, and tiles
def test_gelu_is_as_exact_as_fp32(cuda, M):
    """h = 2^p, p = log2(h): a product of fp32 factors off by 2^-22 of |p| + 1 at most (nine steps, each a rounding that the next ones
    shrink), 2^p by 2^-23; 1 - h by half a step of a value up to 1, and the result's own rounding.  1.7e-8: the fitted p (v h ln 2 times
    its error is 1.6e-8 at most, wherever).  The sum v of a and b is no fp32 number where b is below 2^-16 of a: it is rounded, by 2^-23
    of it at most whichever way, and the result moves by that times the slope of gelu."""
    from promoe_amd import ops
    print(f"case gelu_fp32 M={M}", flush=True)
    n = 4096
    # v = a + b, two bf16 values: the first carries eight bits and the second the next eight
    v = np.concatenate([np.linspace(-14, 14, M * n - 64), np.random.default_rng(1).normal(0, 1e-3, 64)]).reshape(n, M).T.copy().reshape(-1)
    a = torch.from_numpy(v).float().to(torch.bfloat16)
    b = (torch.from_numpy(v) - a.double()).float().to(torch.bfloat16)
    v = (a.double() + b.double()).numpy().reshape(M, n)
    # one row of x against n rows of w: x = (1, 1, 0, ..), w = (a, b, 0, ..); more rows of x: the rows' values by turns
    for m in range(0, M, 50):
        w = torch.zeros(n, 8, dtype=torch.bfloat16)
        w[:, 0], w[:, 1] = a[m * n: (m + 1) * n], b[m * n: (m + 1) * n]
        x = torch.zeros(M, 8, dtype=torch.bfloat16)
        x[:, :2] = 1.0
        y = ops.linear(x.to(cuda), w.to(cuda), act="gelu", out_dtype=torch.float32).double().cpu().numpy()
        assert (y == y[0]).all()
        ref, h = _exact(v[m])
        with np.errstate(divide="ignore"):
            p = np.abs(np.log2(h)) + 1
        tol = np.abs(v[m]) * h * (2.0 ** -23 + 2.0 ** -22 * p * np.log(2)) + np.where(v[m] > 0, np.abs(v[m]) * 2.0 ** -25, 0) \
            + 2.0 ** -24 * np.abs(ref) + 1.7e-8
        slope = np.where(v[m] > 0, 1 - h, h) + v[m] * np.exp(-v[m] ** 2 / 2) / np.sqrt(2 * np.pi)
        tol += 2.0 ** -23 * np.abs(v[m]) * np.abs(slope)
        err = np.abs(y[0] - ref)
        print("  largest error %.2e, of its bound %.2f" % (err.max(), (err / tol).max()), flush=True)
        assert (err <= tol).all()


def test_gelu_far_out(cuda):
    from promoe_amd import ops
    print("case gelu_far", flush=True)
    far = torch.tensor([0.0, 11.0, 13.0, 14.5, 20.0, 100.0, 1e4, 1e10, 1e30, 3e38], dtype=torch.bfloat16)
    v = torch.cat([far, -far]).double()
    w = torch.zeros(20, 8, dtype=torch.bfloat16)
    w[:, 0] = v.to(torch.bfloat16)
    x = torch.zeros(1, 8, dtype=torch.bfloat16)
    x[0, 0] = 1
    y = ops.linear(x.to(cuda), w.to(cuda), act="gelu", out_dtype=torch.float32).double().cpu()[0]
    assert torch.equal(y[:10], v[:10].float().double())
    assert (y[10:] <= 0).all() and (y[10:] > -1e-20).all()
    # (an infinite sum: a product of two large values)
    x[0, 0] = 3e38
    y = ops.linear(x.to(cuda), torch.full((8, 8), 3e38, dtype=torch.bfloat16, device=cuda), act="gelu", out_dtype=torch.float32)
    assert (y == float("inf")).all()
