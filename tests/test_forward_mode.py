"""Forward-mode derivatives (torch.autograd.forward_ad, torch.func.jvp) of the adjacency attention and
the residual norms: like the package's other operators they have none, and say so; a dual tensor does
not require grad, and its tangent must not get lost with the autograd node.  The library's calls are
replaced, nothing is computed."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


@pytest.fixture
def ops(monkeypatch):
    from gnnea import _lib, attention, norm
    from gnnea.graph import DeviceCSR
    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    monkeypatch.setattr(attention, "_forward", lambda q, k, v, csr, meta, want: (q + 0, q))
    monkeypatch.setattr(norm, "_forward", lambda x, y, gate, vecs, meta, want: (x + 0, x + 1, x))
    csr = DeviceCSR(torch.tensor([0, 1], dtype=torch.int32), torch.zeros(1, dtype=torch.int32), None,
                    1, 1)
    return {"attention": lambda x: attention.dot_attention(csr, x, x, x, 1),
            "attention, values": lambda x: attention.dot_attention(csr, torch.ones(1, 4),
                                                                   torch.ones(1, 4), x, 1),
            "residual_norm": lambda x: norm.residual_norm(x, x)[0],
            "weight": lambda x: norm.residual_norm(torch.ones(1, 4), torch.ones(1, 4),
                                                   pre_weight=x[0])[1],
            "norm": lambda x: norm.norm(x)}


@pytest.mark.parametrize("name", ["attention", "attention, values", "residual_norm", "weight", "norm"])
@pytest.mark.parametrize("graph", [True, False])
def test_dual_tensors_are_refused(ops, name, graph):
    x = torch.ones(1, 4)
    with torch.set_grad_enabled(graph):
        with fwd.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError)):
                ops[name](fwd.make_dual(x, x))
            ops[name](x)  # no tangent: as ever
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(ops[name], (x,), (x,))
        assert not ops[name](x).requires_grad
