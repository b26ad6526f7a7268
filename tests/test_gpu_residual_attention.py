"""The adjacency attention, the residual norms and AdamW together, as an encoder and its training
step use them: models.encoders with ``residual`` and ``attention="dot"``, tools/graph_step.py with
``--optim adamw`` / ``adamw8``."""
import types

import numpy as np
import pytest
import torch

from conftest import rel_err

pytestmark = pytest.mark.gpu
# Norm-relative.  The widest chain (a gradient through two blocks) passes four products over 60
# terms, two attention passes and five norms each way: under 30 operators of at most 30 u of their
# terms' absolute sums each (u = 2^-24), sums that cancel by at most a factor of two here: 1e-4.
TOL = 1e-4


def args_of(**kw):
    a = dict(model="GAT", num_layers=3, dim=60, feat_dim=60, act="tanh", dropout=0.0, bias=1,
             n_heads=4, alpha=0.2, n_classes=60, cuda=0, device=torch.device("cuda", 0))
    a.update(kw)
    return types.SimpleNamespace(**a)


def reference(enc, x, mask, heads, kv, kind):
    """The encoder in fp64 with torch's autograd, dense masked softmax."""
    def norm(t, w, b):
        if kind == "layer":
            t = (t - t.mean(1, keepdim=True)) / (t.var(1, unbiased=False, keepdim=True) + 1e-6).sqrt()
        else:
            t = t / (t.pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
        return t * w + (b if b is not None else 0.0)
    P = {k: v.detach().double().cpu().requires_grad_() for k, v in enc.named_parameters()}
    x = x.double().cpu().requires_grad_()

    def get(name, i):
        return P.get("layers.%s.%d" % (name, i))
    r, h = x, norm(x, get("pre_weight", 0), get("pre_bias", 0))
    for i in range(2):
        W = P["layers.blocks.%d.W" % i]
        qkv, d = h @ W, 60 // heads
        outs = []
        for a in range(heads):
            b = a // (heads // kv)
            q = qkv[:, a * d:(a + 1) * d]
            k = qkv[:, (heads + b) * d:(heads + b + 1) * d]
            v = qkv[:, (heads + kv + b) * d:(heads + kv + b + 1) * d]
            s = (q @ k.T / d ** 0.5).masked_fill(~mask, -1e300)
            p = torch.where(mask, torch.softmax(s, 1), torch.zeros_like(s))
            outs.append(p @ v)
        y = torch.tanh(torch.cat(outs, 1))
        n = norm(y, get("post_weight", i), get("post_bias", i))
        g = torch.sigmoid(get("gate", i)) if get("gate", i) is not None else 1.0
        r = r + get("scale", i) * g * n
        h = norm(r, get("pre_weight", i + 1), get("pre_bias", i + 1))
    return x, P, h


@pytest.mark.parametrize("kind,kv,gate", [("rms", 4, False), ("layer", 2, True)])
def test_encoder_against_fp64(device, kind, kv, gate):
    from models.encoders import GAT
    torch.manual_seed(3)
    enc = GAT(args_of(attention="dot", kv_heads=kv, residual=kind, residual_gate=gate)).to(device)
    with torch.no_grad():
        for name, p in enc.named_parameters():
            if "blocks" not in name:
                p.add_(0.2 * torch.randn_like(p))
    n = 90
    g = torch.Generator().manual_seed(1)
    mask = torch.rand(n, n, generator=g) < 0.06
    mask[7] = False
    adj = torch.sparse_coo_tensor(mask.nonzero().T, torch.ones(int(mask.sum())), (n, n)).to(device)
    x = torch.randn(n, 60, generator=g).to(device)
    do = torch.randn(n, 60, generator=g)
    x1 = x.clone().requires_grad_()
    out = enc.encode(x1, adj)
    out.backward(do.to(device))
    x64, P, want = reference(enc, x, mask, 4, kv, kind)
    want.backward(do.double())
    assert rel_err(out.detach().cpu(), want.detach()) < TOL
    assert rel_err(x1.grad.cpu(), x64.grad) < TOL
    for name, p in enc.named_parameters():
        assert rel_err(p.grad.cpu(), P[name].grad) < TOL, name


@pytest.mark.parametrize("model,optim,options", [
    ("GAT", "adamw", dict(attention="dot", residual="layer", kv_heads=2, residual_gate=True)),
    ("GAT", "adamw8", dict(attention="dot", residual="rms")),
    ("HGCN", "adamw", dict(residual="rms")),
    ("GCN", "adamw8", dict())])
def test_ea_iteration_eager_and_replayed(device, model, optim, options):
    """The whole iteration as one graph: losses, gradients and weights equal to the eager step's."""
    from tools.graph_step import run
    p = run(model, 1000, 2500, 5, device, optim, **options)["parity"]
    assert p["loss_rel"] == 0.0 and p["grad_max_rel"] == 0.0 and p["param_max_rel"] == 0.0, p
    assert np.isfinite(p["loss_eager"])


def test_training_steps_against_torch_adam(device):
    """Five steps of a residual attention encoder under AdamW without decay and under torch's Adam:
    the same weights.  An update is at most lr (1 + 21 u) however small the gradient, and Adam's
    first steps magnify a gradient's relative error where the gradient itself is near 0; so the
    gradients are given, not computed, and the weights differ by 21 u lr a step at most, plus
    rounding of the weight: 5 (21 u lr + 2 u |w|)."""
    from gnnea.optim import AdamW
    from models.encoders import GAT
    torch.manual_seed(5)
    enc = GAT(args_of(attention="dot", residual="rms")).to(device)
    ps = [p for p in enc.parameters()]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = AdamW(ps, lr=1e-2, weight_decay=0.0), torch.optim.Adam(qs, lr=1e-2)
    g = torch.Generator(device=device).manual_seed(2)
    for _ in range(5):
        for p, q in zip(ps, qs):
            p.grad = torch.randn(p.shape, generator=g, device=device)
            q.grad = p.grad.clone()
        a.step()
        b.step()
    u = 2.0 ** -24
    for p, q in zip(ps, qs):
        # both sides err
        tol = 2 * 5 * (21 * u * 1e-2 + 2 * u * q.detach().abs())
        assert bool(((p - q).detach().abs() <= tol).all())


def test_sharded_adjacency_is_refused(device):
    from gnnea.dist_graph import DistAdj
    d = DistAdj.__new__(DistAdj)
    d.part, d.engine = types.SimpleNamespace(g=2), None
    with pytest.raises(NotImplementedError):
        d.dot_attention(None, None, None, 1)
