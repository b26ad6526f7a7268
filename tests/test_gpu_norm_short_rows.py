"""gnnea.norm on rows of one to three values, whose gradients are what is left of a difference.

LayerNorm of one value is constant: n = 0, and dy, dx - dr, the weights' gradients and the gate's
share of n are 0, exactly, whatever 1 / sqrt(eps) would make of a rounding.  u = 2^-24.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def run(device, n, D, gate, dtype, seed, kind="layer"):
    from gnnea.norm import residual_norm
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=g).to(dtype).to(device).requires_grad_()  # noqa: E731
    z = dict(none=None, row=lambda: mk(D), full=lambda: mk(n, D))[gate]
    t = dict(x=mk(n, D), y=mk(n, D), z=z and z(), s=mk(D), pw=mk(D), pb=mk(D), qw=mk(D), qb=mk(D))
    dr, dh = mk(n, D).detach(), mk(n, D).detach()
    r, h = residual_norm(*t.values(), kind=kind)
    wrt = [k for k in t if t[k] is not None]
    grads = dict(zip(wrt, torch.autograd.grad((r, h), [t[k] for k in wrt], (dr, dh))))
    return t, dr, dh, r.detach(), h.detach(), grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["none", "row", "full"])
@pytest.mark.parametrize("n", [1, 300])
def test_layer_norm_of_one_value(device, n, gate, dtype):
    t, dr, dh, r, h, grads = run(device, n, 1, gate, dtype, n)
    assert torch.equal(grads["x"], dr)
    for k in ("y", "pw", "qw"):
        assert not grads[k].any(), k
    assert torch.equal(h, t["qb"].detach().expand(n, 1))


@pytest.mark.parametrize("gate", ["none", "row", "full"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("D", [2, 3, 5, 8])
def test_means_and_roots(device, D, kind, gate):
    """The stored statistics, a mean and 1 / deviation, read from norm(x) of rows that make them
    visible: with a weight of 1, h = (x - mean) rho.  mean: D - 1 additions of at most sum|x| each
    rounded, and 0.6 of a last place (1.2 u); rho: half the variance's (D + 3) u and 1.2 u; their
    difference and product 2 u.  (Without the last step of the root and of the mean 3 u each.)"""
    from gnnea.norm import norm
    g = torch.Generator().manual_seed(D)
    x = torch.randn(4000, D, generator=g)
    h = norm(x.to(device), kind=kind).double().cpu()
    x = x.double()
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros(len(x), 1).double()
    rho = 1 / ((x - mean).pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
    off = U * ((D - 1) * x.abs().sum(1, keepdim=True) / D + 1.2 * mean.abs()) * (kind == "layer")
    # (the deviation moves with the mean's error only in second order)
    bound = rho * off + ((D + 3) / 2 + 1.2 + 2) * U * ((x - mean) * rho).abs() + rho * off * off * rho
    assert bool(((h - (x - mean) * rho).abs() <= bound).all())


@pytest.mark.parametrize("D", [3, 300, 700])
def test_squares_that_overflow(device, D):
    """Values whose squares leave fp32: the root mean square is infinite, its reciprocal 0."""
    from gnnea.norm import norm
    x = torch.full((2, D), 1e20, device=device)
    x[1] = 1.0
    h = norm(x, kind="rms")
    assert not h[0].any() and bool(((h[1] - 1).abs() < 1e-6).all())
