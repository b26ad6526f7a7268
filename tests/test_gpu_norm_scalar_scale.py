"""A one-element residual scale in bf16: its gradient is a sum over all columns, rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("D", [300, 1500])
@pytest.mark.parametrize("weights", [True, False])
def test_gradient_of_one_scale_is_rounded_once(device, D, weights):
    """x, y, scale (and weights) in bf16: ds = sum over rows and columns of dx N(y).  The sums are
    fp32: (256 + 64) u of a column's absolute terms, as for a vector's gradients, D more u for the
    columns; then half a step of bf16 of the value.  (A rounding to bf16 per column would err by
    2^-9 of the absolute sum over columns, here 30 to 60 times the value's own size.)"""
    from gnnea.norm import residual_norm
    n = 64
    g = torch.Generator().manual_seed(D)
    x, y, dr = (torch.randn(n, D, generator=g).bfloat16().to(device) for _ in range(3))
    w = (torch.randn(D, generator=g).bfloat16().to(device) if weights else None)
    s = torch.full((1,), 0.5, dtype=torch.bfloat16, device=device, requires_grad=True)
    r, _ = residual_norm(x, y, scale=s, post_weight=w, pre=False)
    ds, = torch.autograd.grad(r, s, dr)
    assert ds.dtype == torch.bfloat16 and ds.shape == (1,)
    y, dr = y.double(), dr.double()
    ny = y / (y.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * (w.double() if weights else 1.0)
    want, size = float((dr * ny).sum()), float((dr * ny).abs().sum())
    assert abs(float(ds) - want) <= (256 + 64 + D) * U * size + 2.0 ** -8 * abs(want)


def test_columns_that_cancel(device):
    """Columns whose sums are 257 and -256 by turns (257 is not a bf16 value, 256 is): 150 are left of
    150 pairs; rounded each to bf16 first, none.  y is all ones, N(y) = 1 / sqrt(1 + 1e-6)."""
    from gnnea.norm import residual_norm
    n, D = 257, 300
    dr = torch.ones(n, D, dtype=torch.bfloat16, device=device)
    dr[:, 1::2] = -1
    dr[0, 1::2] = 0
    y = torch.ones(n, D, dtype=torch.bfloat16, device=device)
    s = torch.ones(1, dtype=torch.bfloat16, device=device, requires_grad=True)
    r, _ = residual_norm(torch.zeros_like(y), y, scale=s, pre=False)
    ds, = torch.autograd.grad(r, s, dr)
    want, size = 150 / (1 + 1e-6) ** 0.5, 300 * 257
    assert abs(float(ds) - want) <= (256 + 64 + D) * U * size + 2.0 ** -8 * want
