"""gnnea_attn_* where rows are very many, and where long rows have no pieces: every row is written."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_long_rows_without_pieces(device):
    """A limit without a list of pieces: rows over it are computed whole (as the C entry allows it)."""
    from gnnea.attention import dot_attention
    from gnnea.graph import DeviceCSR
    g = torch.Generator().manual_seed(0)
    mask = torch.rand(20, 50, generator=g) < 0.5
    q, k, v, do = (torch.randn(n, 8, generator=g).to(device) for n in (20, 50, 50, 20))
    got = []
    for limit in (16, 256):
        row, col = (t.to(device) for t in mask.nonzero().T)
        adj = DeviceCSR.from_coo(row, col, None, 20, 50)
        for a in (adj, adj.transpose()):
            a._attn_pieces = types.SimpleNamespace(limit=limit, n_long=0, n_items=0)
        x = [t.clone().requires_grad_() for t in (q, k, v)]
        out = dot_attention(adj, *x, 2)
        got.append((out.detach(),) + torch.autograd.grad(out, x, do))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_more_rows_than_one_launch_takes(device):
    """2^26 + 5 rows (64 work-items each are over 2^32), entries in a few of them at both ends and
    where a launch ends: as from a small matrix, all other rows 0; as rows and as columns."""
    from gnnea.attention import dot_attention
    from gnnea.graph import DeviceCSR
    n, few, C = 2 ** 26 + 5, 8, 300
    at = torch.tensor([0, 3, 2 ** 25 - 1, 2 ** 25, 2 ** 25 + 1, n - 6, n - 5, n - 1])
    g = torch.Generator().manual_seed(1)
    mask = torch.rand(few, C, generator=g) < 0.1
    mask[3] = True  # in pieces
    row, col = mask.nonzero().T
    far, row, col = at[row].to(device), row.to(device), col.to(device)
    k, v = (torch.randn(C, 4, generator=g).bfloat16().to(device) for _ in range(2))
    qs, ds = (torch.randn(few, 4, generator=g).bfloat16().to(device) for _ in range(2))
    at = at.to(device)

    def wide(t):
        out = torch.zeros(n, 4, dtype=t.dtype, device=device)
        out[at] = t
        return out

    def run(adj, q, k, v, do):
        x = [t.clone().requires_grad_() for t in (q, k, v)]
        out = dot_attention(adj, *x, 1)
        return (out.detach(),) + torch.autograd.grad(out, x, do)
    for few_args, wide_args, big in (
            ((row, col, None, few, C, qs, k, v, ds), (far, col, None, n, C, wide(qs), k, v, wide(ds)), (0, 1)),
            ((col, row, None, C, few, k, qs, ds, v), (col, far, None, C, n, k, wide(qs), wide(ds), v), (2, 3))):
        want = run(DeviceCSR.from_coo(*few_args[:5]), *few_args[5:])
        got = run(DeviceCSR.from_coo(*wide_args[:5]), *wide_args[5:])
        for i, (a, b) in enumerate(zip(got, want)):
            if i not in big:
                assert torch.equal(a, b), i
                continue
            assert torch.equal(a[at], b), i
            a[at] = 0
            assert not a.any(), i
        del got
