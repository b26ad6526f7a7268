"""Norms before and after a block, fused with the block's gate and residual scale (gnnea_norm_*).

One call takes a residual stack from one block's output to the next block's input:

    r = x + scale * sigmoid(gate) * N(y)        y: the block's output, x: the residual stream
    h = N'(r)                                   the next block's input

with N(t) = n weight + bias, n = t / rms(t) (``kind="rms"``) or (t - mean) / deviation
(``kind="layer"``).  The reference's HighWay layer (layers/layers.py:45-80) has the gate and the
residual, without norms or a scale.  Every element is read once and written once in each
direction, statistics and sums are fp32 or wider, results do not change from run to run.
"""
import torch

from . import _lib
from ._lib import NormProblem, check, ptr, stream_of
from .ops import FEATURE_DTYPES, _ld, _rows, needs_node

KINDS = {"rms": _lib.GNNEA_NORM_RMS, "layer": _lib.GNNEA_NORM_LAYER}
MAX_D = 8192


def _code(dtype):
    return _lib.GNNEA_BF16 if dtype == torch.bfloat16 else _lib.GNNEA_F32


def _problem(x, y, gate, vecs, meta):
    kind, eps, post, pre, alpha = meta
    n, D = x.shape
    a = NormProblem(n=n, D=D, dtype=_code(x.dtype), kind=kind, eps=eps, post=post, pre=pre,
                    alpha=alpha, x=x.data_ptr(), ldx=_ld(x))
    w = None
    if y is not None:
        a.y, a.ldy = y.data_ptr(), _ld(y)
    if gate is not None:
        a.gate = gate.data_ptr()
        if gate.dim() == 2:
            a.gate_mode, a.ldg = _lib.GNNEA_GATE_FULL, _ld(gate)
        else:
            a.gate_mode, w = _lib.GNNEA_GATE_ROW, gate
    for name, v in zip(_VECTORS, vecs):
        if v is not None:
            setattr(a, name, v.data_ptr())
            w = v
    a.w_dtype = _lib.GNNEA_F32 if w is None else _code(w.dtype)
    return a


_VECTORS = ("scale", "post_w", "post_b", "pre_w", "pre_b")
_GRADS = ("dscale", "dpost_w", "dpost_b", "dpre_w", "dpre_b")


def _forward(x, y, gate, vecs, meta, want_stats):
    """(r, h, the rows' statistics for a backward pass)."""
    a = _problem(x, y, gate, vecs, meta)
    (n, D), dtype, device = x.shape, x.dtype, x.device
    r = h = stats = None
    if y is not None:
        r = torch.empty((n, D), dtype=dtype, device=device)
        a.r, a.ldr = r.data_ptr(), D
    if meta[3]:
        h = torch.empty((n, D), dtype=dtype, device=device)
        a.h, a.ldh = h.data_ptr(), D
    if want_stats:
        stats = torch.empty((n, 4), dtype=torch.float32, device=device)
        a.stats = stats.data_ptr()
    if n:
        with _lib.on_device(device):
            check(_lib.lib().gnnea_norm_fwd(a, stream_of(device)))
    return r, h, stats


def _grad_rows(t, dtype):
    return t if t.dtype == dtype and t.is_contiguous() else _rows(t, dtype)


class NormFn(torch.autograd.Function):
    """(r, h) of residual_norm; r is None without y, h without the norm of the next block."""

    @staticmethod
    def forward(ctx, x, y, gate, scale, pw, pb, qw, qb, meta):
        vecs = (scale, pw, pb, qw, qb)
        r, h, stats = _forward(x, y, gate, vecs, meta, any(ctx.needs_input_grad))
        ctx.save_for_backward(x, y, gate, scale, pw, pb, qw, qb, stats)
        ctx.meta = meta
        ctx.set_materialize_grads(False)
        return r, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dr, dh):
        x, y, gate, scale, pw, pb, qw, qb, stats = ctx.saved_tensors
        if dr is None and dh is None:
            return (None,) * 9
        vecs, need = (scale, pw, pb, qw, qb), ctx.needs_input_grad
        (n, D), dtype, device = x.shape, x.dtype, x.device
        if n == 0:
            return tuple(torch.zeros_like(t) if t is not None and want else None for t, want in
                         zip((x, y, gate) + vecs + (None,), need))
        # from what is saved, which hooks may have moved since
        a = _problem(x, y, gate, vecs, ctx.meta)
        a.stats = stats.data_ptr()
        if dr is not None:
            dr = _grad_rows(dr, dtype)
            a.dr, a.lddr = dr.data_ptr(), _ld(dr)
        if dh is not None:
            dh = _grad_rows(dh, dtype)
            a.dh, a.lddh = dh.data_ptr(), _ld(dh)
        out = [None] * 9
        a.lddx = a.lddy = a.lddg = D
        if need[0]:
            out[0] = t = torch.empty((n, D), dtype=dtype, device=device)
            a.dx = t.data_ptr()
        if need[1]:
            out[1] = t = torch.empty((n, D), dtype=dtype, device=device)
            a.dy = t.data_ptr()
        sums = any(need[3:8])
        if need[2]:
            rows = gate.dim() == 2
            out[2] = t = torch.empty((n, D), dtype=dtype, device=device) if rows else \
                torch.empty_like(gate)
            a.dgate = t.data_ptr()
            sums = sums or not rows
        L = _lib.lib()
        ws, ws_bytes = None, 0
        if sums:
            # the vectors all have one type
            wanted = [k for k in range(5) if need[3 + k]]
            if wanted:
                like = vecs[wanted[0]]
                got = torch.empty((len(wanted), D), dtype=like.dtype, device=device).unbind(0)
                for k, t in zip(wanted, got):
                    out[3 + k] = t
                    setattr(a, _GRADS[k], t.data_ptr())
            ws_bytes = int(L.gnnea_norm_bwd_ws_bytes(n, D, a.dtype))
            ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=device)
        with _lib.on_device(device):
            check(L.gnnea_norm_bwd(a, ptr(ws), ws_bytes, stream_of(device)))
        return tuple(out)


def _matrix(name, t, x):
    if t.dtype != x.dtype or t.device != x.device or t.shape != x.shape:
        raise ValueError("gnnea.norm: %s must be like x: %s %s on %s (got %s %s on %s)"
                         % (name, tuple(x.shape), x.dtype, x.device, tuple(t.shape), t.dtype,
                            t.device))
    return _rows(t)


def _vectors(x, names, vecs):
    """The vectors in one type: x's, or fp32 where they are mixed or fp32 already."""
    D = x.shape[1]
    for name, v in zip(names, vecs):
        if v is None:
            continue
        if v.dim() != 1 or v.shape[0] != D or v.dtype not in FEATURE_DTYPES or \
                v.device != x.device:
            raise ValueError("gnnea.norm: %s must be a vector of %d fp32 or bf16 values on %s "
                             "(got %s %s on %s)" % (name, D, x.device, tuple(v.shape), v.dtype,
                                                    v.device))
    types = {v.dtype for v in vecs if v is not None}
    if len(types) > 1 or (x.dtype == torch.float32 and torch.bfloat16 in types):
        vecs = [None if v is None else v.float() for v in vecs]
    return [None if v is None else v.contiguous() for v in vecs]


def _features(x):
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or not 1 <= x.shape[1] <= MAX_D:
        raise ValueError("gnnea.norm: x must be [N, D] with 1 <= D <= %d" % MAX_D)
    if x.dtype not in FEATURE_DTYPES:
        raise TypeError("gnnea.norm: fp32 or bf16 features required (got %s)" % x.dtype)


def _kind(kind, eps):
    if kind not in KINDS:
        raise ValueError("gnnea.norm: kind must be 'rms' or 'layer' (got %r)" % (kind,))
    if not eps > 0:
        raise ValueError("gnnea.norm: eps must be positive (got %r)" % (eps,))
    return KINDS[kind]


def _apply(x, y, gate, vecs, meta):
    if needs_node(x, y, gate, *vecs):
        return NormFn.apply(x, y, gate, *vecs, meta)
    return _forward(x, y, gate, vecs, meta, False)[:2]


def residual_norm(x, y, gate=None, scale=None, post_weight=None, post_bias=None, pre_weight=None,
                  pre_bias=None, kind="rms", eps=1e-6, post=True, pre=True):
    """(r, h): r = x + scale * sigmoid(gate) * N(y), h = N'(r).

    x, y        [N, D] fp32 or bf16, the residual stream and the block's output
    gate        pre-activations [N, D], or [D] for all rows, or None (no gate)
    scale       a number, a vector [D] or a one-element tensor (residual scale), or None (1)
    post_*      weight and bias [D] of the norm N after the block; ``post=False``: N(y) = y
    pre_*       weight and bias [D] of the norm N' before the next block; ``pre=False``: h is None
    Vectors are fp32 or of x's type; without a weight (bias) it is 1 (0).  D <= 8192.  Gradients
    for every tensor argument, of its own type and shape."""
    _features(x)
    _lib.require_device(x, y, gate, *(t for t in (scale, post_weight, post_bias, pre_weight,
                                                 pre_bias) if isinstance(t, torch.Tensor)))
    code = _kind(kind, eps)
    if not post and (post_weight is not None or post_bias is not None):
        raise ValueError("gnnea.residual_norm: post=False takes no post_weight or post_bias")
    if not pre and (pre_weight is not None or pre_bias is not None):
        raise ValueError("gnnea.residual_norm: pre=False takes no pre_weight or pre_bias")
    alpha = 1.0
    if scale is not None and not isinstance(scale, torch.Tensor):
        alpha, scale = float(scale), None
    elif scale is not None and scale.numel() == 1:
        if scale.dtype == torch.bfloat16:  # its gradient, a sum over columns, is then rounded once
            scale = scale.float()
        scale = scale.reshape(1).expand(x.shape[1])
    y = _matrix("y", y, x)
    names = ("scale", "post_weight", "post_bias", "pre_weight", "pre_bias", "gate")
    row_gate = gate if gate is not None and gate.dim() == 1 else None
    *vecs, row_gate = _vectors(x, names, (scale, post_weight, post_bias, pre_weight, pre_bias,
                                          row_gate))
    if gate is not None:
        gate = row_gate if row_gate is not None else _matrix("gate", gate, x)
    return _apply(_rows(x), y, gate, vecs, (code, float(eps), int(post), int(pre), alpha))


def norm(x, weight=None, bias=None, kind="rms", eps=1e-6):
    """N(x) alone (the first block's input of a residual stack, or its last output)."""
    _features(x)
    _lib.require_device(x, weight, bias)
    code = _kind(kind, eps)
    weight, bias = _vectors(x, ("weight", "bias"), (weight, bias))
    return _apply(_rows(x), None, None, (None, None, None, weight, bias),
                  (code, float(eps), 0, 1, 1.0))[1]
