"""Dot-product attention over a sparse adjacency (gnnea_attn_*), beside ops.gat's additive scores
(layers/att_layers.py:29-61).

    o_i = sum_c p_ic v_c,   p_ic = softmax over the stored entries c of row i of (scale q_i . k_c)

for all heads at once, key/value heads shared by groups of query heads.  Nothing per entry is
stored: the backward pass recomputes the probabilities from the row's log-sum-exp, once over the
matrix (dq) and once over its transpose (dk, dv).
"""
import torch

from . import _lib
from ._lib import AttnProblem, check, ptr, stream_of
from .graph import csr_of
from .ops import FEATURE_DTYPES, _ld, _rows, needs_node

MAX_D_HEAD = 256
# rows with more stored entries are cut into pieces of as many, one wave each
LONG_ROW = 256


class _Pieces:
    """The pieces of a CSR's long rows (they depend on rowptr alone; built once per matrix)."""

    def __init__(self, csr):
        deg, limit = csr.degrees().long(), LONG_ROW
        rows = torch.nonzero(deg > limit).flatten()  # one setup sync
        self.limit = limit
        self.n_long = int(rows.numel())
        self.n_items = 0
        self.rows = self.ptr = self.items = None
        if self.n_long:
            count = (deg[rows] + limit - 1) // limit
            end = torch.cumsum(count, 0)
            self.n_items = int(end[-1])
            which = torch.repeat_interleave(torch.arange(self.n_long, device=rows.device), count)
            slot = torch.arange(self.n_items, device=rows.device)
            row = rows[which]
            beg = csr.rowptr[row].long() + (slot - (end - count)[which]) * limit
            stop = torch.minimum(beg + limit, csr.rowptr[row + 1].long())
            self.items = torch.stack([row, beg, stop, slot], 1).to(torch.int32).contiguous()
            self.rows = rows.to(torch.int32)
            self.ptr = torch.cat([end.new_zeros(1), end]).to(torch.int32)
            # kept with the matrix, so the next call may come on another stream
            torch.cuda.current_stream(csr.device).synchronize()


def _pieces(csr):
    if getattr(csr, "_attn_pieces", None) is None:
        csr._attn_pieces = _Pieces(csr)
    return csr._attn_pieces


def _problem(csr, q, k, v, meta):
    heads, kv_heads, scale = meta
    pieces = _pieces(csr)
    a = AttnProblem()
    a.rowptr = csr.rowptr.data_ptr()
    a.col = (csr.col if csr.nnz else csr.rowptr).data_ptr()  # without entries: never read
    a.n_rows, a.n_cols = csr.n_rows, csr.n_cols
    a.heads, a.kv_heads, a.d_head, a.scale = heads, kv_heads, q.shape[1] // heads, scale
    a.dtype = _lib.GNNEA_BF16 if q.dtype == torch.bfloat16 else _lib.GNNEA_F32
    a.limit = pieces.limit
    if pieces.n_long:
        a.n_items, a.n_long = pieces.n_items, pieces.n_long
        a.items, a.long_rows, a.long_ptr = (t.data_ptr() for t in (pieces.items, pieces.rows,
                                                                  pieces.ptr))
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.ldq, a.ldk, a.ldv = _ld(q), _ld(k), _ld(v)
    return a


def _run(which, a, device):
    L = _lib.lib()
    ws, ws_bytes = None, 0
    if a.n_items:
        ws_bytes = int(L.gnnea_attn_ws_bytes(a, which))
        ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=device)
    fn = (L.gnnea_attn_fwd, L.gnnea_attn_bwd_rows, L.gnnea_attn_bwd_cols)[which]
    with _lib.on_device(device):
        check(fn(a, ptr(ws), ws_bytes, stream_of(device)))


def _forward(q, k, v, csr, meta, want_lse):
    """(out, lse): lse, the rows' log-sum-exp, for a backward pass."""
    a = _problem(csr, q, k, v, meta)
    out = torch.empty((q.shape[0], q.shape[1]), dtype=q.dtype, device=q.device)
    a.o, a.ldo = out.data_ptr(), q.shape[1]
    lse = None
    if want_lse:
        lse = torch.empty((q.shape[0], meta[0]), dtype=torch.float32, device=q.device)
        a.lse = lse.data_ptr()
    _run(_lib.GNNEA_ATTN_FWD, a, q.device)
    return out, lse


class DotAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, csr, meta):
        out, lse = _forward(q, k, v, csr, meta, any(ctx.needs_input_grad))
        ctx.save_for_backward(q, k, v, lse)
        ctx.csr, ctx.meta = csr, meta
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, lse = ctx.saved_tensors
        dout = _rows(dout, q.dtype)
        need = ctx.needs_input_grad
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        stat = torch.empty((q.shape[0], ctx.meta[0], 2), dtype=torch.float32, device=q.device)
        a = _problem(ctx.csr, q, k, v, ctx.meta)  # from what is saved, which hooks may have moved
        a.lse, a.stat = lse.data_ptr(), stat.data_ptr()
        a.dout, a.lddo = dout.data_ptr(), _ld(dout)
        a.dq, a.lddq = dq.data_ptr(), q.shape[1]
        _run(_lib.GNNEA_ATTN_BWD_ROWS, a, q.device)
        dk = dv = None
        if need[1] or need[2]:
            dk = torch.empty(k.shape, dtype=k.dtype, device=q.device)
            dv = torch.empty(v.shape, dtype=v.dtype, device=q.device)
            a = _problem(ctx.csr.transpose(), q, k, v, ctx.meta)
            a.stat, a.dout, a.lddo = stat.data_ptr(), dout.data_ptr(), _ld(dout)
            a.dk, a.lddk, a.dv, a.lddv = dk.data_ptr(), k.shape[1], dv.data_ptr(), v.shape[1]
            _run(_lib.GNNEA_ATTN_BWD_COLS, a, q.device)
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None,
                None, None)


def dot_attention(adj, q, k, v, heads, kv_heads=None, scale=None):
    """Attention of the rows of ``adj`` over their stored entries; [n_rows, heads * d_head].

    adj     a DeviceCSR or a torch sparse COO tensor [n_rows, n_cols] (its values are not used; an
            entry stored twice counts once)
    q       [n_rows, heads * d_head]; k, v: [n_cols, kv_heads * d_head], fp32 or bf16, columns of
            a wider row-major matrix (one projection for all three) as they are
    kv_heads    key/value heads (None: heads); query head h reads key/value head
            h // (heads / kv_heads)
    scale   None: 1 / sqrt(d_head)
    A row without stored entries, or whose scores are all -inf, gives 0 and passes no gradient;
    rows of k and v that no entry names are never read (and get zero gradients)."""
    _lib.require_device(q, k, v)
    csr = csr_of(adj)
    kv_heads = heads if kv_heads is None else kv_heads
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError("gnnea.dot_attention: heads must be a multiple of kv_heads (got %r, %r)"
                         % (heads, kv_heads))
    dtype, device, d = q.dtype, csr.device, 0
    for name, t, n, h in (("q", q, csr.n_rows, heads), ("k", k, csr.n_cols, kv_heads),
                          ("v", v, csr.n_cols, kv_heads)):
        shape = t.shape
        if len(shape) != 2 or shape[0] != n or shape[1] == 0 or shape[1] % h or \
                (d and shape[1] != h * d):
            raise ValueError("gnnea.dot_attention: %s must be [%d, %d * d_head] (got %s)"
                             % (name, n, h, tuple(shape)))
        d = shape[1] // h
        if t.dtype != dtype or dtype not in FEATURE_DTYPES:
            raise TypeError("gnnea.dot_attention: q, k and v must all be fp32 or all bf16 (got %s)"
                            % t.dtype)
        if t.device != device:
            raise ValueError("gnnea.dot_attention: %s is on %s, the adjacency on %s"
                             % (name, t.device, device))
    if d > MAX_D_HEAD:
        raise ValueError("gnnea.dot_attention: d_head must be at most %d (got %d)"
                         % (MAX_D_HEAD, d))
    meta = (heads, kv_heads, d ** -0.5 if scale is None else float(scale))
    q, k, v = _rows(q), _rows(k), _rows(v)
    if _ld(k) != _ld(v):  # the kernels form one row offset for both
        k, v = k.contiguous(), v.contiguous()
    if needs_node(q, k, v):
        return DotAttentionFn.apply(q, k, v, csr, meta)
    return _forward(q, k, v, csr, meta, False)[0]
