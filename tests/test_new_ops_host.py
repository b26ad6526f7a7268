"""The C-ABI of the adjacency attention, the residual norms and AdamW on the host: struct layouts,
refusals before any launch, and the loud refusal of host tensors."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT

EINVAL, EWORKSPACE, EALIGN = -1, -2, -3


@pytest.fixture(scope="module")
def L():
    from gnnea import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libgnnea.so not built")
    return _lib.lib()


def test_struct_layouts(tmp_path):
    """Every field of the ctypes mirrors at the offset that a C compiler gives it."""
    from gnnea import _lib
    mirrors = dict(gnnea_norm=_lib.NormProblem, gnnea_adamw_tensor=_lib.AdamwTensor,
                   gnnea_attn=_lib.AttnProblem)
    lines = []
    for name, m in mirrors.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        for f, _ in m._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, f, name, f))
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gnnea.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0; }\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", exe, str(src)], check=True)
    got = dict(line.split() for line in subprocess.run([exe], capture_output=True, text=True,
                                                       check=True).stdout.splitlines())
    for name, m in mirrors.items():
        assert int(got[name]) == ctypes.sizeof(m)
        for f, _ in m._fields_:
            assert int(got["%s.%s" % (name, f)]) == getattr(m, f).offset, (name, f)


def norm_problem(**kw):
    from gnnea._lib import NormProblem
    a = NormProblem(n=4, D=8, eps=1e-6, alpha=1.0, post=1, pre=1, x=64, y=64, r=64, h=64, ldx=8,
                    ldy=8, ldr=8, ldh=8, stats=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(n=-1), EINVAL), (dict(D=0), EINVAL), (dict(D=8193), EINVAL), (dict(dtype=1), EINVAL),
    (dict(w_dtype=2), EINVAL), (dict(kind=2), EINVAL), (dict(gate_mode=3), EINVAL),
    (dict(gate_mode=1), EINVAL), (dict(gate=64), EINVAL), (dict(eps=0.0), EINVAL),
    (dict(x=None), EINVAL), (dict(ldx=7), EINVAL), (dict(ldy=7), EINVAL), (dict(r=None), EINVAL),
    (dict(h=None), EINVAL), (dict(y=None), EINVAL), (dict(post=0, post_w=64), EINVAL),
    (dict(pre=0, pre_w=64), EINVAL), (dict(y=None, post=0, pre=0), EINVAL),
    (dict(gate_mode=1, gate=64, ldg=7), EINVAL), (dict(stats=72), EALIGN), (dict(n=0), 0)])
def test_norm_refusals(L, kw, rc):
    assert L.gnnea_norm_fwd(norm_problem(**kw), None) == rc


def test_norm_backward_refusals(L):
    assert L.gnnea_norm_bwd(norm_problem(stats=None), None, 0, None) == EINVAL
    assert L.gnnea_norm_bwd(norm_problem(dr=64, lddr=7), None, 0, None) == EINVAL
    assert L.gnnea_norm_bwd(norm_problem(pre=0, dh=64, lddh=8), None, 0, None) == EINVAL
    assert L.gnnea_norm_bwd(norm_problem(dx=64, lddx=7), None, 0, None) == EINVAL
    need = L.gnnea_norm_bwd_ws_bytes(4, 8, 0)
    assert need > 0 and L.gnnea_norm_bwd_ws_bytes(4, 0, 0) == EINVAL
    ok = norm_problem(dscale=64)
    assert L.gnnea_norm_bwd(ok, 64, need - 1, None) == EWORKSPACE
    assert L.gnnea_norm_bwd(ok, None, need, None) == EINVAL
    assert L.gnnea_norm_bwd(ok, 72, need, None) == EALIGN
    assert L.gnnea_norm_bwd_ws_bytes(10 ** 9, 8192, 2) < 1 << 30  # bounded, whatever the rows


def attn_problem(**kw):
    from gnnea._lib import AttnProblem
    a = AttnProblem(rowptr=64, col=64, n_rows=4, n_cols=4, heads=4, kv_heads=2, d_head=8,
                    scale=1.0, q=64, k=64, v=64, ldq=32, ldk=16, ldv=16, o=64, ldo=32, lse=64,
                    dout=64, lddo=32, stat=64, dq=64, dk=64, dv=64, lddq=32, lddk=16, lddv=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(n_rows=-1), EINVAL), (dict(heads=3), EINVAL), (dict(kv_heads=0), EINVAL),
    (dict(d_head=0), EINVAL), (dict(d_head=257), EINVAL), (dict(dtype=1), EINVAL),
    (dict(scale=float("nan")), EINVAL), (dict(rowptr=None), EINVAL), (dict(col=None), EINVAL),
    (dict(q=None), EINVAL), (dict(k=None), EINVAL), (dict(ldq=31), EINVAL), (dict(ldk=15), EINVAL),
    (dict(ldv=15), EINVAL), (dict(n_items=1), EINVAL), (dict(limit=-1), EINVAL),
    (dict(items=8), EALIGN),
    (dict(n_items=1, n_long=1, limit=4, items=64, long_rows=64, long_ptr=64), EWORKSPACE)])
def test_attention_refusals(L, kw, rc):
    for fn in (L.gnnea_attn_fwd, L.gnnea_attn_bwd_rows, L.gnnea_attn_bwd_cols):
        assert fn(attn_problem(**kw), None, 0, None) == rc, fn
    assert L.gnnea_attn_fwd(attn_problem(n_rows=0), None, 0, None) == 0


def test_attention_pass_refusals(L):
    assert L.gnnea_attn_fwd(attn_problem(o=None), None, 0, None) == EINVAL
    assert L.gnnea_attn_fwd(attn_problem(ldo=31), None, 0, None) == EINVAL
    for kw in (dict(lse=None), dict(dq=None), dict(lddq=31), dict(dout=None), dict(stat=None)):
        assert L.gnnea_attn_bwd_rows(attn_problem(**kw), None, 0, None) == EINVAL
    assert L.gnnea_attn_bwd_rows(attn_problem(stat=68), None, 0, None) == EALIGN
    for kw in (dict(dk=None), dict(dv=None), dict(lddk=15), dict(lddo=31)):
        assert L.gnnea_attn_bwd_cols(attn_problem(**kw), None, 0, None) == EINVAL
    a = attn_problem(n_items=3)
    assert L.gnnea_attn_ws_bytes(a, 0) == 3 * 4 * 10 * 4
    assert L.gnnea_attn_ws_bytes(a, 3) == EINVAL


def test_adamw_refusals(L):
    from gnnea._lib import AdamwTensor
    t = (AdamwTensor * 2)(AdamwTensor(p=64, g=64, m=64, v=64, n=40000), AdamwTensor(n=0))
    step = lambda a=t, c=2, d=0, b=32, ctl=64: L.gnnea_adamw_step(  # noqa: E731
        a, c, d, b, 0.9, 0.999, 1e-8, 0.0, ctl, None)
    assert L.gnnea_adamw_norm_parts(t, 2) == 3
    assert step(b=16) == EINVAL and step(d=1) == EINVAL and step(ctl=None) == EINVAL
    assert step(ctl=68) == EALIGN and step(a=None) == EINVAL and step(c=-1) == EINVAL
    assert step(b=8) == EINVAL  # no scales
    assert L.gnnea_adamw_step(t, 2, 0, 32, 1.0, 0.999, 1e-8, 0.0, 64, None) == EINVAL
    assert L.gnnea_adamw_norm(t, 2, 0, 64, 2, None) == EWORKSPACE
    assert L.gnnea_adamw_begin(None, 1, 1.0, 0.9, 0.999, 1e-3, None, 0, 64, 64, None) == EINVAL
    assert L.gnnea_adamw_begin(None, 0, 0.0, 0.9, 0.999, 1e-3, None, 0, None, 64, None) == EINVAL
    assert L.gnnea_adamw_begin(None, 0, 0.0, 0.9, 0.999, 1e-3, None, 0, 68, 64, None) == EALIGN
    t[0].n = -1
    assert step() == EINVAL and L.gnnea_adamw_norm_parts(t, 2) == EINVAL
    assert step(a=(AdamwTensor * 1)(), c=1) == 0 and step(c=0) == 0


def test_host_tensors_are_refused():
    from gnnea import GnneaError
    from gnnea.attention import dot_attention
    from gnnea.norm import norm, residual_norm
    from gnnea.optim import AdamW
    x = torch.zeros(4, 8)
    with pytest.raises(GnneaError):
        norm(x)
    with pytest.raises(GnneaError):
        residual_norm(x, x)
    with pytest.raises(GnneaError):
        dot_attention(torch.eye(4).to_sparse(), x, x, x, 2)
    p = torch.nn.Parameter(x)
    p.grad = x
    with pytest.raises(GnneaError):
        AdamW([p]).step()


@pytest.mark.parametrize("option", [dict(lr=-1.0), dict(lr=torch.ones(1)), dict(eps=0.0),
                                    dict(weight_decay=-1e-3), dict(betas=(0.9, 1.0)),
                                    dict(betas=(0.9,))])
def test_adamw_options_of_a_group(option):
    """A group's own options are held to the same rules, and a refused group leaves no trace."""
    from gnnea.optim import AdamW
    p, q, r = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    with pytest.raises(ValueError):
        AdamW([dict(params=[p], **option)])
    with pytest.raises(ValueError):
        AdamW([p], **option)
    opt = AdamW([p, q])
    for bad in (dict(params=[r], **option), dict(params=[p, r])):  # the second: p is there already
        with pytest.raises(ValueError):
            opt.add_param_group(bad)
        assert len(opt.param_groups) == 1 and opt._base == [0]
    with pytest.raises(TypeError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(3).double())]))
    opt.add_param_group(dict(params=[r]))
    assert opt._base == [0, 2]


def encoder_args(**kw):
    import types
    a = dict(num_layers=3, dim=12, feat_dim=12, act="relu", dropout=0.0, bias=1, n_heads=4,
             alpha=0.2, cuda=-1, device="cpu")
    a.update(kw)
    return types.SimpleNamespace(**a)


def test_encoder_options():
    """Without the options the encoders are what they were; with them, residual stacks and
    dot-product layers with parameters of these names and shapes."""
    from layers.att_layers import DotAttentionLayer
    from layers.layers import ResidualStack
    from models.encoders import GAT, GCN, HGCN, MLP
    for cls in (GCN, GAT, HGCN, MLP):
        assert isinstance(cls(encoder_args()).layers, torch.nn.Sequential)
    assert isinstance(MLP(encoder_args(residual="rms")).layers, torch.nn.Sequential)
    enc = GAT(encoder_args(attention="dot", kv_heads=2, residual="layer", residual_gate=True))
    assert isinstance(enc.layers, ResidualStack)
    assert isinstance(enc.layers.blocks[0], DotAttentionLayer)
    sd = enc.state_dict()
    assert sd["layers.blocks.1.W"].shape == (12, (4 + 2 * 2) * 3)
    assert {"layers.pre_weight.2", "layers.pre_bias.2", "layers.post_weight.1", "layers.post_bias.1",
            "layers.scale.1", "layers.gate.1"} <= set(sd)
    assert "layers.gate.0" not in GCN(encoder_args(residual="rms")).state_dict()
    with pytest.raises(ValueError):
        GCN(encoder_args(residual="rms", feat_dim=10))
    with pytest.raises(ValueError):
        GCN(encoder_args(residual="batch"))
    with pytest.raises(ValueError):
        DotAttentionLayer(12, 3, 0.0, torch.relu, 4, True, kv_heads=3)
