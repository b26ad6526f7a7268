"""gnnea.norm against fp64 formulas, every gradient included.

Tolerances.  u = 2^-24.  A row's sums go through at most 16 values per thread, 6 cross-lane adds
and 7 waves, so a sum is off by at most 32 u of its terms' absolute sum, a mean or 1 / rms by 40 u;
the longest chain of an output (dy) is two statistics, the recomputed residual row, a dot product
over the row and some 30 products: under 256 u of the sum of the absolute terms it is made of,
which `scales` forms in fp64 (each factor by its absolute value, each normalised value n by
|n| + mean|t| rho: the subtraction of the mean).  Column sums add rows: at most 64 more.  Then eps
/ 2 of the value for the one rounding of the output's type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
K = 256
NAMES = ("x", "y", "gate", "scale", "pw", "pb", "qw", "qb")


def reference(t, kind, alpha, post, pre, dr, dh, eps=1e-6):
    """fp64 (r, h, gradients) and the absolute scales of each."""
    t = {k: (None if v is None else v.double().cpu()) for k, v in t.items()}
    x, y, z, s, w, b, w2, b2 = (t[k] for k in NAMES)
    dr, dh = (None if g is None else g.double().cpu() for g in (dr, dh))
    D = x.shape[1]
    one = torch.ones(D).double()

    def stats(v):
        mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros(len(v), 1).double()
        rho = 1 / ((v - mean).pow(2).mean(1, keepdim=True) + eps).sqrt()
        n = (v - mean) * rho
        return n, rho, n.abs() + v.abs().mean(1, keepdim=True) * rho

    def back(q, n, rho, qa, na):
        m = q - n * (q * n).mean(1, keepdim=True)
        ma = qa + na * (qa * na).mean(1, keepdim=True)
        if kind == "layer":
            m = m - q.mean(1, keepdim=True)
            ma = ma + qa.mean(1, keepdim=True)
        return rho * m, rho * ma

    w_, w2_, s_ = (one if v is None else v for v in (w, w2, s))
    out, sc = {}, {}
    if y is not None:
        n, rho, na = stats(y) if post else (y, torch.ones(len(y), 1).double(), y.abs())
        a, aa = n * w_, na * w_.abs()
        if b is not None:
            a, aa = a + b, aa + b.abs()
        g = torch.sigmoid(z) if z is not None else one.expand_as(y)
        r, ra = x + alpha * s_ * g * a, x.abs() + abs(alpha) * s_.abs() * g * aa
        out["r"], sc["r"] = r, ra
    else:
        r, ra = x, x.abs()
    dx, dxa = (torch.zeros_like(x),) * 2 if dr is None else (dr, dr.abs())
    if pre:
        n2, rho2, n2a = stats(r)
        n2a = n2a + ra * rho2  # n' moves with r's own error
        out["h"], sc["h"] = n2 * w2_, n2a * w2_.abs()
        if b2 is not None:
            out["h"], sc["h"] = out["h"] + b2, sc["h"] + b2.abs()
        if dh is not None:
            d, da_ = back(dh * w2_, n2, rho2, dh.abs() * w2_.abs(), n2a)
            dx, dxa = dx + d, dxa + da_
            out["qw"], sc["qw"] = (dh * n2).sum(0), (dh.abs() * n2a).sum(0)
            out["qb"], sc["qb"] = dh.sum(0), dh.abs().sum(0)
    out["x"], sc["x"] = dx, dxa
    if y is not None:
        da, daa = dx * alpha * s_ * g, dxa * abs(alpha) * s_.abs() * g
        d, e = back(da * w_, n, rho, daa * w_.abs(), na) if post else (da, daa)
        out["y"], sc["y"] = d, e
        dz, dza = da * a * (1 - g), daa * aa * (1 - g)
        if z is not None:
            rows = z.dim() == 1
            out["gate"], sc["gate"] = (dz.sum(0), dza.sum(0)) if rows else (dz, dza)
        out["scale"], sc["scale"] = (alpha * dx * g * a).sum(0), (abs(alpha) * dxa * g * aa).sum(0)
        out["pw"], sc["pw"] = (da * n).sum(0), (daa * na).sum(0)
        out["pb"], sc["pb"] = da.sum(0), daa.sum(0)
    return out, sc


def inputs(n, D, dtype, wdtype, gate, device, seed, layer=True, scale=True):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s, t=dtype: torch.randn(s, generator=g).to(t).to(device)  # noqa: E731
    t = dict(x=mk(n, D), y=mk(n, D) * 2 + 0.5, gate=None, scale=mk(D, t=wdtype) if scale else None,
             pw=mk(D, t=wdtype), pb=mk(D, t=wdtype) if layer else None, qw=mk(D, t=wdtype),
             qb=mk(D, t=wdtype) if layer else None)
    if gate == "full":
        t["gate"] = mk(n, D) * 3
    elif gate == "row":
        t["gate"] = mk(D, t=wdtype)
    return t, mk(n, D), mk(n, D)


def run(t, kind, dr, dh, post=True, pre=True, alpha=None):
    from gnnea.norm import residual_norm
    t = {k: (None if v is None else v.detach().requires_grad_()) for k, v in t.items()}
    r, h = residual_norm(t["x"], t["y"], t["gate"], t["scale"] if alpha is None else alpha,
                         t["pw"], t["pb"], t["qw"], t["qb"], kind=kind, post=post, pre=pre)
    outs = [(o, g) for o, g in ((r, dr), (h, dh)) if o is not None and g is not None]
    names = [k for k in NAMES if t[k] is not None and (alpha is None or k != "scale")]
    grads = torch.autograd.grad([o for o, _ in outs], [t[k] for k in names], [g for _, g in outs],
                                allow_unused=True)
    got = {k: g for k, g in zip(names, grads) if g is not None}
    got.update(r=r.detach())
    if h is not None:
        got["h"] = h.detach()
    return got


def compare(got, want, scales, t):
    for name, g in got.items():
        w, s = want[name], scales[name]
        assert tuple(g.shape) == tuple(w.shape), name
        assert g.dtype == t.get(name, t["x"]).dtype, name
        tol = (K + 64) * U * s + torch.finfo(g.dtype).eps / 2 * w.abs() + 1e-37
        worst = float(((g.double().cpu() - w).abs() / tol).max())
        assert worst <= 1.0, (name, worst)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32),
                                          (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("n,D,gate", [
    (1, 1, "full"), (3, 1, "row"), (1, 300, "none"), (5, 3, "full"), (130, 17, "row"),
    (70, 64, "full"), (67, 300, "full"), (40, 301, "row"), (33, 1023, "full"), (9, 1025, "none"),
    (6, 2049, "full"), (5, 4097, "row"), (3, 8191, "full"), (2, 8192, "none"), (5000, 75, "full")])
def test_against_fp64(device, n, D, gate, kind, dtype, wdtype):
    t, dr, dh = inputs(n, D, dtype, wdtype, gate, device, n + D, kind == "layer")
    got = run(t, kind, dr, dh)
    want, scales = reference(t, kind, 1.0, True, True, dr, dh)
    compare(got, want, scales, t)


@pytest.mark.parametrize("post,pre,alpha,use", [
    (False, True, 0.25, "both"), (True, False, None, "r"), (False, False, -1.5, "r"),
    (True, True, None, "r"), (True, True, None, "h")])
def test_parts(device, post, pre, alpha, use):
    """Without either norm, with a constant scale, with gradients for one output alone."""
    t, dr, dh = inputs(50, 300, torch.float32, torch.float32, "full", device, 4)
    if not post:
        t["pw"] = t["pb"] = None
    if not pre:
        t["qw"] = t["qb"] = None
    if alpha is not None:
        t["scale"] = None
    dr, dh = (dr if use != "h" else None), (dh if use != "r" else None)
    got = run(t, "layer", dr, dh, post, pre, alpha)
    want, scales = reference(t, "layer", 1.0 if alpha is None else alpha, post, pre, dr, dh)
    if use == "r" and pre:  # h takes no part: its vectors have no gradient to compare
        got = {k: v for k, v in got.items() if k not in ("qw", "qb")}
    compare(got, want, scales, t)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norm_alone(device, kind):
    from gnnea.norm import norm
    t, _, dh = inputs(77, 300, torch.bfloat16, torch.float32, "none", device, 5, kind == "layer")
    x, w, b = (None if v is None else v.detach().requires_grad_() for v in (t["x"], t["qw"], t["qb"]))
    h = norm(x, w, b, kind=kind)
    wrt = [v for v in (x, w, b) if v is not None]
    grads = torch.autograd.grad(h, wrt, dh)
    t["y"] = None
    want, scales = reference(t, kind, 1.0, False, True, None, dh)
    got = dict(zip(("x", "qw", "qb"), grads), h=h.detach())
    compare(got, want, scales, t)


def test_strided_broadcast_and_scalar_scale(device):
    """Column blocks of wider buffers, an expanded row, a one-element scale: its gradient is the
    sum over columns of the vector's."""
    from gnnea.norm import residual_norm
    t, dr, dh = inputs(40, 60, torch.float32, torch.float32, "full", device, 6)
    wide = torch.randn(40, 131, device=device)
    wide[:, 3:63] = t["x"]
    base = run(t, "layer", dr, dh)
    t2 = dict(t, x=wide[:, 3:63], y=t["y"].t().contiguous().t())
    got = run(t2, "layer", dr.t().contiguous().t(), dh)
    for k in base:
        assert torch.equal(base[k], got[k]), k
    one = torch.full((1,), 0.5, device=device, requires_grad=True)
    r, h = residual_norm(t["x"], t["y"], None, one, kind="rms")
    ds, = torch.autograd.grad((r, h), one, (dr, dh))
    vec = torch.full((60,), 0.5, device=device, requires_grad=True)
    r2, h2 = residual_norm(t["x"], t["y"], None, vec, kind="rms")
    dv, = torch.autograd.grad((r2, h2), vec, (dr, dh))
    assert torch.equal(r, r2) and ds.shape == (1,)
    assert abs(float(ds) - float(dv.double().sum())) <= 64 * U * float(dv.abs().sum())
    row = torch.randn(1, 60, device=device).expand(40, 60)
    r3, _ = residual_norm(row, t["y"], pre=False, kind="rms")
    assert torch.equal(r3, residual_norm(row.contiguous(), t["y"], pre=False, kind="rms")[0])


def test_extremes_and_no_rows(device):
    """A constant row (variance 0), a row of zeros, NaN in one row only, zero rows."""
    from gnnea.norm import norm, residual_norm
    x = torch.zeros(4, 300, device=device)
    x[1] = 3.0
    x[2] = torch.randn(300, device=device)
    x[3, 7] = float("nan")
    h = norm(x, kind="layer")
    assert not h[:2].any() and bool(torch.isfinite(h[2]).all()) and bool(torch.isnan(h[3]).all())
    w = torch.ones(300, device=device, requires_grad=True)
    e = torch.zeros(0, 300, device=device, requires_grad=True)
    r, h = residual_norm(e, e, scale=w, pre_weight=w)
    assert r.shape == h.shape == (0, 300)
    gw, ge = torch.autograd.grad((r, h), (w, e), (torch.zeros_like(r), torch.zeros_like(h)))
    assert not gw.any() and ge.shape == (0, 300)


def test_differences(device):
    """Directional derivatives against central differences of the outputs (h = 1e-2: third
    derivatives are of order 1 along a unit direction, 1e-4; rounding 1e-7 * norm / h)."""
    from gnnea.norm import residual_norm
    t, dr, dh = inputs(20, 48, torch.float32, torch.float32, "full", device, 8)
    got = run(t, "layer", dr, dh)
    g = torch.Generator().manual_seed(2)
    h = 1e-2
    for name in NAMES:
        d = torch.randn(t[name].shape, generator=g).to(device)
        d /= d.norm()
        f = []
        for s in (h, -h):
            u = dict(t)
            u[name] = t[name] + s * d
            r, hh = residual_norm(u["x"], u["y"], u["gate"], u["scale"], u["pw"], u["pb"], u["qw"],
                                  u["qb"], kind="layer")
            f.append(float((r.double() * dr).sum() + (hh.double() * dh).sum()))
        diff, mine = (f[0] - f[1]) / (2 * h), float((got[name].double() * d).sum())
        size = float(dr.norm() + dh.norm())
        assert abs(diff - mine) < 1e-4 * size + 1e-7 * size * 10 / h, (name, diff, mine)


def test_captured_replays_and_stream(device):
    from gnnea.norm import residual_norm
    t, dr, dh = inputs(500, 300, torch.bfloat16, torch.float32, "row", device, 9)
    leaf = {k: (None if v is None else v.requires_grad_()) for k, v in t.items()}
    names = [k for k in NAMES if leaf[k] is not None]

    def step():
        r, h = residual_norm(*(leaf[k] for k in NAMES), kind="layer")
        return (r, h) + torch.autograd.grad((r, h), [leaf[k] for k in names], (dr, dh))
    s = torch.cuda.Stream(device)
    s.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream(device).wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    for it in range(4):
        with torch.no_grad():
            for k in names:
                leaf[k].mul_(0.9)
        g, res = graphs[it % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, step()):
            assert torch.equal(a, b)


def test_refusals(device):
    from gnnea.norm import norm, residual_norm
    x = torch.randn(4, 8, device=device)
    w = torch.ones(8, device=device)
    for kw in (dict(kind="group"), dict(eps=0.0), dict(post=False, post_weight=w),
               dict(pre=False, pre_bias=w), dict(gate=torch.ones(4, 1, device=device)),
               dict(gate=torch.ones(7, device=device)), dict(scale=torch.ones(7, device=device)),
               dict(post_weight=w.double())):
        with pytest.raises(ValueError):
            residual_norm(x, x, **kw)
    with pytest.raises(ValueError):
        residual_norm(x, x[:3])
    with pytest.raises(ValueError):
        residual_norm(x, x.bfloat16())
    with pytest.raises(TypeError):
        norm(x.half())
    with pytest.raises(ValueError):
        norm(torch.ones(2, 8193, device=device))
    with pytest.raises(ValueError):
        norm(torch.ones(2, 3, 8, device=device))


def test_offsets_past_32_bits(device):
    """8M rows of 300 (2.4e9 elements): the last rows as from a small call, column sums of a
    constant exact (every sum of the call is a whole number below 2^24)."""
    from gnnea.norm import residual_norm
    n, D = 8_000_000, 300
    x = torch.zeros(n, D, dtype=torch.bfloat16, device=device)
    y = torch.ones(n, D, dtype=torch.bfloat16, device=device)
    g = torch.Generator().manual_seed(0)
    x[-70:] = torch.randn(70, D, generator=g).bfloat16().to(device)
    y[-70:] = torch.randn(70, D, generator=g).bfloat16().to(device)
    w = torch.ones(D, device=device)
    r, h = residual_norm(x, y, scale=0.5, post_weight=w, pre_weight=w)
    r2, h2 = residual_norm(x[-70:], y[-70:], scale=0.5, post_weight=w, pre_weight=w)
    assert torch.equal(r[-70:], r2) and torch.equal(h[-70:], h2)
    del r, h
    b = torch.zeros(D, device=device, requires_grad=True)
    y.requires_grad_()
    r, _ = residual_norm(x, y, post_weight=w, post_bias=b, pre=False, kind="layer")
    dr = torch.ones(1, 1, dtype=torch.bfloat16, device=device).expand(n, D).contiguous()
    db, dy = torch.autograd.grad(r, (b, y), dr)
    assert bool((db == n).all())
    assert bool((dy[-70:].float().abs() <= 2.0 ** -8).all())  # a constant's gradient through N is 0


def test_the_same_tensor_twice(device):
    """residual_norm(x, x): the gradient is the sum of both arguments' gradients."""
    from gnnea.norm import residual_norm
    t, dr, dh = inputs(30, 300, torch.float32, torch.float32, "none", device, 11)
    x = t["x"].clone().requires_grad_()
    r, h = residual_norm(x, x, scale=0.5, kind="layer")
    got, = torch.autograd.grad((r, h), x, (dr, dh))
    a, b = (t["x"].clone().requires_grad_() for _ in range(2))
    r2, h2 = residual_norm(a, b, scale=0.5, kind="layer")
    ga, gb = torch.autograd.grad((r2, h2), (a, b), (dr, dh))
    assert torch.equal(r, r2) and torch.equal(got, ga + gb)


def test_saved_tensors_that_move(device):
    """Saved tensors packed to the host and back (other addresses, other strides): the same bits."""
    from gnnea.norm import residual_norm
    t, dr, dh = inputs(40, 60, torch.float32, torch.float32, "full", device, 13)
    wide = torch.zeros(40, 200, device=device)
    wide[:, 5:65] = t["x"]
    t["x"] = wide[:, 5:65]
    want = run(t, "layer", dr, dh)
    leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
    with torch.autograd.graph.save_on_cpu():
        r, h = residual_norm(*(leaf[k] for k in NAMES), kind="layer")
    junk = [torch.full((40, 60), 7.0, device=device) for _ in range(8)]
    got = torch.autograd.grad((r, h), [leaf[k] for k in NAMES], (dr, dh))
    del junk
    for k, g in zip(NAMES, got):
        assert torch.equal(g, want[k]), k
