"""gnnea.attention.dot_attention against a dense fp64 restatement of its formulas.

Tolerances.  u = 2^-24 (fp32), t = eps / 2 of the output's type.  A score is a dot product of d
terms, so it is off by at most e_s = (d + 6) u scale sum|q||k| (products, sums, the two factors of
scale and log2 e, the reference of the exponent); a probability relatively by e_p = 2 max e_s +
(n + 16) u, n the row's entries (its sum, exp2's last place, the rescaling by the running maximum).
Then, with D = max |dp| of the row and e_d = (d + 2) u max sum|do||v|,
    |o|   e_p + (n + 8) u of sum p|v|
    ds    p (3 e_p D + 3 e_d + (n + 8) u 2 D)      (delta = sum p dp, subtracted)
    dq    scale sum_c (that) |k| + (n + 8) u scale sum |ds||k|
and dk, dv the same over columns; each plus t of the value for its one rounding.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def dense(mask, q, k, v, do, heads, kv, scale):
    """(values, bounds) of out, dq, dk, dv in fp64; mask [R, C]."""
    R, C = mask.shape
    d = q.shape[1] // heads
    q, k, v, do = (t.double().cpu() for t in (q, k, v, do))
    mask = mask.cpu()
    n = mask.sum(1).double()
    out, dq = torch.zeros(R, heads * d).double(), torch.zeros(R, heads * d).double()
    dk, dv = torch.zeros(C, kv * d).double(), torch.zeros(C, kv * d).double()
    bo, bq, bk, bv = (torch.zeros_like(t) for t in (out, dq, dk, dv))
    ncol = mask.sum(0).double()[:, None]
    for h in range(heads):
        a, b = slice(h * d, (h + 1) * d), slice(h // (heads // kv) * d, (h // (heads // kv) + 1) * d)
        qh, kh, vh, dh = q[:, a], k[:, b], v[:, b], do[:, a]
        kh, vh = kh.nan_to_num(0.0, 0.0, 0.0), vh.nan_to_num(0.0, 0.0, 0.0)  # rows nobody names
        s = (qh @ kh.T * scale).masked_fill(~mask, -math.inf)
        top = s.amax(1, keepdim=True) if C else torch.zeros(R, 1).double()
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = torch.exp(s - top)
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
        p = torch.where(mask, p, torch.zeros_like(p))
        dp = dh @ vh.T
        ds = p * (dp - (p * dp).sum(1, keepdim=True))
        out[:, a], dq[:, a] = p @ vh, ds @ kh * scale
        dk[:, b] += ds.T @ qh * scale
        dv[:, b] += p.T @ dh
        es = (d + 6) * U * scale * (qh.abs() @ kh.abs().T * mask).amax(1) if C else torch.zeros(R)
        ep = (2 * es + (n + 16) * U)[:, None]
        big = (dp.abs() * mask).amax(1, keepdim=True) if C else torch.zeros(R, 1)
        ed = (d + 2) * U * (dh.abs() @ vh.abs().T * mask).amax(1, keepdim=True) if C else 0
        eds = p * (3 * ep * big + 3 * ed + (n[:, None] + 8) * U * 2 * big)
        bo[:, a] = (ep + (n[:, None] + 8) * U) * (p @ vh.abs())
        bq[:, a] = scale * (eds @ kh.abs() + (n[:, None] + 8) * U * (2 * p * big) @ kh.abs())
        share = heads // kv
        bk[:, b] += scale * (eds.T @ qh.abs()
                             + (ncol * share + 8) * U * ((2 * p * big).T @ qh.abs()))
        bv[:, b] += (p * ep).T @ dh.abs() + (ncol * share + 8) * U * (p.T @ dh.abs())
    return (out, dq, dk, dv), (bo, bq, bk, bv)


def check(got, want, bound, t):
    for name, g, w, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
        assert g.shape == w.shape and bool(torch.isfinite(g).all()), name
        err = (g.double().cpu() - w).abs()
        tol = b + t * w.abs() + 1e-37
        worst = float((err / tol).max()) if err.numel() else 0.0
        assert worst <= 1.0, (name, worst)


def csr(device, mask):
    from gnnea.graph import DeviceCSR
    row, col = torch.nonzero(mask).T.contiguous()
    return DeviceCSR.from_coo(row.to(device), col.to(device), None, *mask.shape)


def case(R, C, heads, kv, d, dtype, per_row, device, seed=0, fused=False):
    g = torch.Generator().manual_seed(seed)
    mask = torch.rand(R, C, generator=g) < per_row / max(C, 1)
    if R > 4:
        mask[1] = False       # a row without entries
        mask[R - 1] = False
        mask[2] = True        # a row with all
        mask[:, C // 2] = False  # a column that nobody names
    wq, wk = heads * d, kv * d
    mk = lambda n, w: torch.randn(n, w, generator=g).to(dtype).to(device)  # noqa: E731
    if fused and R == C:
        x = mk(R, wq + 2 * wk)
        q, k, v = x[:, :wq], x[:, wq:wq + wk], x[:, wq + wk:]
    else:
        q, k, v = mk(R, wq), mk(C, wk), mk(C, wk)
    if R > 4:
        for t in (k, v):      # never read
            t[C // 2] = float("nan")
    return mask, q, k, v, mk(R, wq)


def both(adj, q, k, v, do, heads, kv, scale=None):
    from gnnea.attention import dot_attention
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = dot_attention(adj, q, k, v, heads, kv, scale)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), do)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,C,heads,kv,d,per_row,fused", [
    (1, 1, 1, 1, 1, 2, False),        # one row, one entry, one value
    (1, 7, 2, 1, 3, 4, False),
    (37, 37, 4, 4, 75, 5, True),      # the encoders' heads; columns of one projection
    (65, 40, 8, 2, 32, 9, False),     # shared key/value heads, another number of columns
    (33, 50, 6, 2, 20, 7, False),     # three heads share one; heads not a power of two
    (20, 20, 9, 3, 17, 6, True),      # more heads than a wave has groups
    (40, 40, 1, 1, 128, 3, False),
    (30, 30, 2, 2, 256, 4, True),     # the widest head
    (24, 24, 3, 1, 5, 4, True),       # heads narrower than 16 bytes
    (24, 24, 2, 2, 131, 4, True),
    (64, 64, 16, 16, 16, 6, False),
    (300, 700, 4, 2, 33, 3, False),   # row 2 has 699 entries: cut into pieces
    (700, 300, 2, 1, 64, 3, False),   # (its columns too, in the transposed matrix)
])
def test_against_fp64(device, dtype, R, C, heads, kv, d, per_row, fused):
    mask, q, k, v, do = case(R, C, heads, kv, d, dtype, per_row, device, R + d, fused)
    if C == 300:
        mask[3:R - 1, 5] = True  # a column that nearly all rows name
    got = both(csr(device, mask), q, k, v, do, heads, kv)
    want, bound = dense(mask, q, k, v, do, heads, kv, d ** -0.5)
    check(got, want, bound, torch.finfo(dtype).eps / 2)
    if R > 4:
        assert not got[0][1].any() and not got[1][1].any()           # the empty row
        assert not got[2][C // 2].any() and not got[3][C // 2].any()  # the unnamed column


def test_pieces_equal_whole_rows_in_value(device, monkeypatch):
    """Cut at 256 or at 16 entries: the same values within the bounds, and a second run the same
    bits."""
    from gnnea import attention
    mask, q, k, v, do = case(50, 600, 4, 4, 24, torch.float32, 40, device)
    want, bound = dense(mask, q, k, v, do, 4, 4, 24 ** -0.5)
    for cut in (256, 16, 100000):
        monkeypatch.setattr(attention, "LONG_ROW", cut)
        adj = csr(device, mask)
        got = both(adj, q, k, v, do, 4, 4)
        check(got, want, bound, torch.finfo(torch.float32).eps / 2)
        for a, b in zip(got, both(adj, q, k, v, do, 4, 4)):
            assert torch.equal(a, b)


def test_gradient_against_differences(device):
    """Directional derivative of sum(out * R): central differences of the operator's own outputs.
    With step h the difference is off by h^2 / 6 of the third derivative (about 10 h^2 here) and
    by the outputs' rounding, about 1e-7 sqrt(sum R^2 n d) / h."""
    from gnnea.attention import dot_attention
    mask, q, k, v, do = case(40, 40, 4, 2, 16, torch.float32, 6, device, 3)
    adj = csr(device, mask)
    k, v = k.nan_to_num(), v.nan_to_num()
    got = both(adj, q, k, v, do, 4, 2)
    g = torch.Generator().manual_seed(9)
    h = 1e-2
    for i in range(3):
        t = [q, k, v]
        dirn = torch.randn(t[i].shape, generator=g).to(device)
        dirn /= dirn.norm()
        f = []
        for s in (h, -h):
            t2 = list(t)
            t2[i] = t[i] + s * dirn
            f.append(float((dot_attention(adj, *t2, 4, 2).double() * do.double()).sum()))
        diff = (f[0] - f[1]) / (2 * h)
        mine = float((got[1 + i].double() * dirn.double()).sum())
        assert abs(diff - mine) < 10 * h * h + 1e-7 * float(do.norm()) * 4 / h, (i, diff, mine)


def test_large_and_infinite_scores(device):
    """Scores of +-1e4 (a softmax without its shift overflows) and keys of -inf: a row all of
    whose scores are -inf gives zero and no gradient, like one without entries."""
    from gnnea.attention import dot_attention
    mask = torch.ones(3, 4, dtype=torch.bool)
    q = torch.full((3, 8), 100.0, device=device)
    q[1] = -100.0
    k = torch.randn(4, 8, generator=torch.Generator().manual_seed(0)).to(device) * 12
    v = torch.randn(4, 8, generator=torch.Generator().manual_seed(1)).to(device)
    do = torch.ones(3, 8, device=device)
    got = both(csr(device, mask), q, k, v, do, 1, 1, 1.0)
    want, bound = dense(mask, q, k, v, do, 1, 1, 1.0)
    check(got, want, bound, U)
    mask = torch.tensor([[True, True], [False, True]])
    q = torch.ones(2, 4, device=device)
    k = torch.tensor([[0.5] * 4, [-math.inf] * 4], device=device)
    v = torch.tensor([[2.0] * 4, [3.0] * 4], device=device)
    out = dot_attention(csr(device, mask), q, k, v, 1)
    assert torch.equal(out.cpu(), torch.tensor([[2.0] * 4, [0.0] * 4]))


def test_empty_matrix_and_coo_adjacency(device):
    from gnnea.attention import dot_attention
    from gnnea.graph import DeviceCSR
    none = torch.zeros(0, dtype=torch.int64, device=device)
    adj = DeviceCSR.from_coo(none, none, None, 5, 3)
    q = torch.randn(5, 8, device=device)
    k = torch.randn(3, 8, device=device)
    for t in both(adj, q, k, k.clone(), torch.ones_like(q), 2, 2):
        assert not t.any()
    idx = torch.tensor([[0, 0, 1, 1], [1, 1, 0, 2]], device=device)  # an entry stored twice
    coo = torch.sparse_coo_tensor(idx, torch.ones(4, device=device), (2, 3))
    out = dot_attention(coo, q[:2], k, k, 2)
    mask = torch.tensor([[False, True, False], [True, False, True]])
    want, bound = dense(mask, q[:2], k, k, torch.ones(2, 8), 2, 2, 0.5)
    check((out,), want[:1], bound[:1], U)


def test_other_stream_and_partial_gradients(device):
    from gnnea.attention import dot_attention
    mask, q, k, v, do = case(50, 50, 4, 2, 24, torch.bfloat16, 6, device)
    adj = csr(device, mask)
    want = both(adj, q, k, v, do, 4, 2)
    s = torch.cuda.Stream(device)
    s.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(s):
        got = both(adj, q, k, v, do, 4, 2)
    torch.cuda.current_stream(device).wait_stream(s)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    v2 = v.detach().requires_grad_()
    out = dot_attention(adj, q, k, v2, 4, 2)
    assert torch.equal(torch.autograd.grad(out, v2, do)[0], want[3])


def test_first_calls_on_two_streams(device):
    """What is kept with a matrix is written before the call that makes it returns."""
    from gnnea.attention import _pieces
    mask, q, k, v, do = case(40, 3000, 2, 1, 16, torch.float32, 3, device, 4)
    adj, again = csr(device, mask), csr(device, mask)
    want = both(csr(device, mask), q, k, v, do, 2, 1)
    torch.cuda.synchronize()
    pieces = _pieces(adj)
    assert torch.cuda.current_stream(device).query() and pieces.n_long
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    got = []
    for s in streams:  # the second does not wait for the first
        with torch.cuda.stream(s):
            got.append(both(again, q, k, v, do, 2, 1))
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(want, g):
            assert torch.equal(a, b)


def test_captured_and_replayed(device):
    """Two graphs of one matrix, replayed in turn with eager work between: both read new inputs."""
    from gnnea.attention import dot_attention
    mask, q, k, v, do = case(300, 700, 4, 2, 16, torch.float32, 4, device, 5)
    adj = csr(device, mask)
    q, k, v = (t.nan_to_num().requires_grad_() for t in (q, k, v))
    s = torch.cuda.Stream(device)
    s.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(dot_attention(adj, q, k, v, 4, 2), (q, k, v), do)
    torch.cuda.current_stream(device).wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = dot_attention(adj, q, k, v, 4, 2)
            res = (out,) + torch.autograd.grad(out, (q, k, v), do)
        graphs.append((g, res))
    for it in range(4):
        with torch.no_grad():
            for t in (q, k, v, do):
                t.mul_(0.9).add_(0.01 * (it + 1))
        g, res = graphs[it % 2]
        g.replay()
        torch.cuda.synchronize()
        want = both(adj, q, k, v, do, 4, 2)
        for a, b in zip(res, want):
            assert torch.equal(a.detach(), b)


def test_refusals(device):
    from gnnea.attention import dot_attention
    mask, q, k, v, _ = case(10, 10, 2, 2, 8, torch.float32, 4, device)
    adj = csr(device, mask)
    for bad in (dict(heads=3), dict(heads=2, kv_heads=3), dict(heads=0), dict(heads=4, kv_heads=4, k=k[:, :8])):
        args = dict(q=q, k=k, v=v, heads=2)
        args.update(bad)
        with pytest.raises(ValueError):
            dot_attention(adj, **args)
    with pytest.raises(ValueError):
        dot_attention(adj, q[:9], k, v, 2)
    with pytest.raises(TypeError):
        dot_attention(adj, q, k.bfloat16(), v, 2)
    with pytest.raises(TypeError):
        dot_attention(adj, q.half(), k.half(), v.half(), 2)
    wide = torch.zeros(10, 257, device=device)
    with pytest.raises(ValueError):
        dot_attention(adj, wide, wide, wide, 1)
    with pytest.raises(RuntimeError):
        qq = q.clone().requires_grad_()
        gq, = torch.autograd.grad(dot_attention(adj, qq, k, v, 2).sum(), qq, create_graph=True)
        gq.sum().backward()


def test_offsets_past_32_bits(device):
    """Keys and values whose elements lie past 2^32 in their buffer (17M rows, 256 apart): the same
    bits as from a small buffer."""
    from gnnea.attention import dot_attention
    from gnnea.graph import DeviceCSR
    n, ld = 17_000_000, 256
    wide = torch.zeros(n, ld, dtype=torch.bfloat16, device=device)
    g = torch.Generator().manual_seed(4)
    cols = torch.tensor([0, 5, n - 300, n - 2, n - 1])
    kv = torch.randn(5, 32, generator=g).bfloat16().to(device)
    wide[cols.to(device), :32] = kv
    row = torch.tensor([0, 0, 1, 1, 1, 2])
    pick = torch.tensor([0, 3, 1, 2, 4, 4])
    q = torch.randn(3, 16, generator=g).bfloat16().to(device)
    do = torch.randn(3, 16, generator=g).bfloat16().to(device)
    far = DeviceCSR.from_coo(row.to(device), cols[pick].to(device), None, 3, n)
    near = DeviceCSR.from_coo(row.to(device), pick.to(device), None, 3, 5)
    out = dot_attention(far, q, wide[:, :16], wide[:, 16:32], 2)
    assert torch.equal(out, dot_attention(near, q, kv[:, :16], kv[:, 16:], 2))
    # queries past 2^32: the transposed matrix gathers them
    back = DeviceCSR.from_coo(cols[pick].to(device), row.to(device), None, n, 3)
    small = DeviceCSR.from_coo(pick.to(device), row.to(device), None, 5, 3)
    Q = wide[:, :16].detach().requires_grad_()
    D = torch.zeros(n, 16, dtype=torch.bfloat16, device=device)
    D[cols.to(device)] = kv[:, 16:]
    k = q.clone().requires_grad_()
    got = torch.autograd.grad(dot_attention(back, Q, k, do, 2), (Q, k), D)
    Qs, ks = kv[:, :16].detach().clone().requires_grad_(), q.clone().requires_grad_()
    want = torch.autograd.grad(dot_attention(small, Qs, ks, do, 2), (Qs, ks), kv[:, 16:].contiguous())
    assert torch.equal(got[1], want[1]) and torch.equal(got[0][cols.to(device)], want[0])


@pytest.mark.parametrize("R,C", [(0, 4), (4, 0), (0, 0)])
def test_no_rows_or_columns(device, R, C):
    from gnnea.graph import DeviceCSR
    none = torch.zeros(0, dtype=torch.int64, device=device)
    adj = DeviceCSR.from_coo(none, none, None, R, C)
    q, k = torch.ones(R, 8, device=device), torch.ones(C, 4, device=device)
    out, dq, dk, dv = both(adj, q, k, k.clone(), torch.ones_like(q), 2, 1)
    assert out.shape == dq.shape == (R, 8) and dk.shape == dv.shape == (C, 4)
    assert not out.any() and not dq.any() and not dk.any() and not dv.any()


def test_shared_leaves_and_frozen_inputs(device):
    """One tensor as q, k and v gets the sum of the three gradients; without a gradient wanted the
    outputs are the same bits."""
    from gnnea.attention import dot_attention
    mask, q, _, _, do = case(30, 30, 2, 2, 16, torch.float32, 5, device, 8)
    adj = csr(device, mask)
    x = q.clone().requires_grad_()
    out = dot_attention(adj, x, x, x, 2)
    got, = torch.autograd.grad(out, x, do)
    parts = both(adj, q, q.clone(), q.clone(), do, 2, 2)
    assert torch.equal(out.detach(), parts[0]) and torch.equal(out.detach(), dot_attention(adj, q, q, q, 2))
    # the engine adds the three in an order of its own: two roundings of the sum
    want = parts[1].double() + parts[2].double() + parts[3].double()
    bound = 2 * U * (parts[1].abs() + parts[2].abs() + parts[3].abs()).double()
    assert bool(((got.double() - want).abs() <= bound + 1e-37).all())


def test_saved_tensors_that_move(device):
    """Saved tensors packed to the host and back (other addresses, other strides): the same bits."""
    from gnnea.attention import dot_attention
    mask, q, k, v, do = case(40, 40, 4, 2, 24, torch.float32, 6, device, 12, fused=True)
    adj = csr(device, mask)
    want = both(adj, q, k, v, do, 4, 2)
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    with torch.autograd.graph.save_on_cpu():
        out = dot_attention(adj, *x, 4, 2)
    junk = [torch.full((40, 192), 7.0, device=device) for _ in range(8)]
    got = torch.autograd.grad(out, x, do)
    del junk
    for a, b in zip(want[1:], got):
        assert torch.equal(a, b)
