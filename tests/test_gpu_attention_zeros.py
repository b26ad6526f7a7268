"""Gradients of gnnea.attention.dot_attention where the softmax has none, or little.

ds = p (dp - delta), delta = sum p dp: what all dp of a row have in common does not count.  Where a
row has one entry, or entries whose values are the same, dq and dk are 0, exactly: dp - delta is a
difference of equal numbers.  Otherwise the error goes by the differences of a row's dp, not by
their size (bounds at the test).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SHAPES = [(1, 1, 8), (4, 4, 75), (8, 2, 32), (6, 2, 20), (3, 1, 5), (2, 2, 131), (2, 1, 256)]


def both(device, row, col, R, C, q, k, v, do, heads, kv, scale=None):
    from gnnea.attention import dot_attention
    from gnnea.graph import DeviceCSR
    adj = DeviceCSR.from_coo(row.to(device), col.to(device), None, R, C)
    x = [t.to(device).requires_grad_() for t in (q, k, v)]
    out = dot_attention(adj, *x, heads, kv, scale)
    return (out.detach(),) + torch.autograd.grad(out, x, do.to(device))


def normal(dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return lambda n, w, by=1.0: (torch.randn(n, w, generator=g) * by).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,d", SHAPES)
@pytest.mark.parametrize("n,C", [(1, 1), (9, 9), (700, 700), (700, 3)])
def test_rows_of_one_entry(device, n, C, heads, kv, d, dtype):
    """Self loops, and many rows on few columns (long rows of the transposed matrix), large scores and
    large dp: the output is the value itself, dq and dk are 0."""
    mk = normal(dtype, n + d)
    row = torch.arange(n)
    col = row % C
    q, k, v, do = mk(n, heads * d, 20.0), mk(C, kv * d), mk(C, kv * d), mk(n, heads * d, 1e4)
    out, dq, dk, _ = both(device, row, col, n, C, q, k, v, do, heads, kv)
    want = v.view(C, kv, 1, d).expand(C, kv, heads // kv, d).reshape(C, heads * d)[col]
    assert torch.equal(out.cpu(), want)
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,d", SHAPES)
def test_rows_of_equal_values(device, heads, kv, d, dtype):
    """Many entries, cut into pieces where they are over 256, all of one value row."""
    R, C = 21, 700
    mk = normal(dtype, d)
    mask = torch.rand(R, C, generator=torch.Generator().manual_seed(d)) < 0.02
    mask[2], mask[3] = True, False
    mask[4, :300] = True
    row, col = mask.nonzero().T
    q, k, do = mk(R, heads * d), mk(C, kv * d), mk(R, heads * d, 1e4)
    v = mk(1, kv * d).expand(C, kv * d).contiguous()
    _, dq, dk, _ = both(device, row, col, R, C, q, k, v, do, heads, kv)
    assert not dq.any() and not dk.any()


def exact(mask, q, k, v, do, scale):
    """(dq, dk) of one head in fp64, and a row's quantities for the bounds."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    s = (q @ k.T * scale).masked_fill(~mask, -torch.inf)
    p = torch.softmax(s, 1)
    dp = do @ v.T
    ds = p * (dp - (p * dp).sum(1, keepdim=True))
    return ds @ k * scale, ds.T @ q * scale, p, dp


@pytest.mark.parametrize("C", [40, 700])
def test_values_with_much_in_common(device, C):
    """dp = 1e4 plus differences of order 1.  u = 2^-24, n a row's entries, d the terms of a score.
    dp is off by at most e_d = (d + 2) u sum |do||v|, the one error that goes by its size; p relatively
    by e_p = (2 d + 12) u max(scale sum |q||k|) + (n + 16) u.  With D = max |dp - dp'| of the row, the
    reference among its dp, a term of ds is off by at most p (3 e_p D + 4 e_d + (n + 8) u 2 D), the
    sums over entries by (n + 8) u of their terms p D |k|, over rows by (R + 8) u likewise."""
    R, d, scale = 30, 16, 0.25
    g = torch.Generator().manual_seed(C)
    q, k = torch.randn(R, d, generator=g), torch.randn(C, d, generator=g)
    do = torch.ones(R, d) + 0.01 * torch.randn(R, d, generator=g)
    v = 625.0 + torch.randn(C, d, generator=g) / 4
    mask = torch.rand(R, C, generator=g) < 10 / C
    mask[:, 0] = True
    mask[5] = True  # (700: in pieces)
    row, col = mask.nonzero().T
    _, dq, dk, _ = both(device, row, col, R, C, q, k, v, do, 1, 1, scale)
    wq, wk, p, dp = exact(mask, q, k, v, do, scale)
    q, k, v, do = (t.double() for t in (q, k, v, do))
    n = mask.sum(1, keepdim=True).double()
    far = torch.where(mask, dp, dp[:, :1])
    D = far.amax(1, keepdim=True) - far.amin(1, keepdim=True)
    ep = (2 * d + 12) * U * scale * (q.abs() @ k.abs().T * mask).amax(1, keepdim=True) + (n + 16) * U
    ed = (d + 2) * U * (do.abs() @ v.abs().T)
    eds = p * (3 * ep * D + 4 * ed + (n + 8) * U * 2 * D)
    bq = scale * (eds @ k.abs() + (n + 8) * U * (p * 2 * D) @ k.abs()) + U * wq.abs()
    bk = scale * (eds.T @ q.abs() + (R + 8) * U * (p * 2 * D).T @ q.abs()) + U * wk.abs()
    assert bool(((dq.double().cpu() - wq).abs() <= bq).all())
    assert bool(((dk.double().cpu() - wk).abs() <= bk).all())


def test_exact_differences_of_large_numbers(device):
    """dp = 2^20 + 0 .. 63, exact in fp32 in any order of its sums (whole numbers under 2^24), so
    only differences err: by p (3 e_p D + (n + 8) u 2 D) and the sums as above, D = 63.  Rows of 700
    entries, in pieces; the rounding of sums of p 2^20 |k| would be 2^20 / 63 times as large."""
    R, C, d, scale = 6, 700, 8, 0.25
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(R, d, generator=g), torch.randn(C, d, generator=g)
    do = torch.ones(R, d)
    v = torch.full((C, d), 2.0 ** 17)
    v[:, 0] += torch.randint(0, 64, (C,), generator=g)
    mask = torch.ones(R, C, dtype=torch.bool)
    row, col = mask.nonzero().T
    _, dq, dk, _ = both(device, row, col, R, C, q, k, v, do, 1, 1, scale)
    wq, wk, p, _ = exact(mask, q, k, v, do, scale)
    q, k = q.double(), k.double()
    ep = (2 * d + 12) * U * scale * (q.abs() @ k.abs().T).amax(1, keepdim=True) + (C + 16) * U
    eds = p * 63 * (3 * ep + (C + 8) * U * 2)
    bq = scale * (eds @ k.abs() + (C + 8) * U * 126 * p @ k.abs()) + U * wq.abs()
    # (dk subtracts delta = c + e, rounded at the size of c: half a step of 2^20, an eighth)
    bk = scale * ((eds + p * 2.0 ** -4).T @ q.abs() + (R + 8) * U * 126 * p.T @ q.abs()) + U * wk.abs()
    assert bool(((dq.double().cpu() - wq).abs() <= bq).all())
    assert bool(((dk.double().cpu() - wk).abs() <= bk).all())


@pytest.mark.parametrize("first", [True, False])
def test_a_large_value_without_weight(device, first):
    """An entry of weight e^-60 whose dp is 1e6 times the others', at either end of its row, leaves
    the row's dq as it is without it: its own part is 1e6 e^-60 < 1e-19.  c is then another entry's
    dp, |dp - c| <= 2 D with D = max |dp| of the others, so both sides err by the e_p and sums of
    above: (e_p + (n + 16) u) sum p 2 D |k|, e_p = (2 d + 12) u max sum |q||k| + (n + 16) u, and by
    dp's own rounding, (d + 2) u sum |do||v|."""
    n, d = 12, 8
    g = torch.Generator().manual_seed(3)
    q, k = torch.ones(1, d), torch.randn(n, d, generator=g) / 4
    v, do = torch.randn(n, d, generator=g), torch.randn(1, d, generator=g)
    at = 0 if first else n - 1
    k[at], v[at] = -60.0 / d, v[at] * 1e6
    rest = torch.tensor([i for i in range(n) if i != at])
    args = device, torch.zeros(n, dtype=torch.long), torch.arange(n), 1, n, q, k, v, do, 1, 1, 1.0
    less = args[:1] + (args[1][1:], rest) + args[3:]
    got, want = both(*args)[1].cpu(), both(*less)[1].cpu()
    q, k, v, do = (t.double() for t in (q, k[rest], v[rest], do))
    p, dp = torch.softmax(q @ k.T, 1), do @ v.T
    ep = (2 * d + 12) * U * float((q.abs() @ k.abs().T).max()) + (n + 16) * U
    ed = (d + 2) * U * (do.abs() @ v.abs().T)
    bound = 2 * (p * ((ep + (n + 16) * U) * 2 * dp.abs().max() + 4 * ed)) @ k.abs()
    assert bool(((got - want).abs().double() <= bound).all())
