"""AdamW over many tensors in few launches, moments in 32 or 8 bits (gnnea_adamw_*).

The reference trains with torch.optim.Adam (run/train_ea.py:28-34); ``AdamW`` takes its place in
the same loop (``weight_decay=0`` is Adam), with the gradients' global norm clipped in the same
step where ``max_norm`` is given.  The step counter and the learning rate stay on the device, so a
step can be captured into a HIP graph as it is.
"""
from array import array

import torch

from . import _lib
from ._lib import check, stream_of
from .ops import FEATURE_DTYPES

BLOCK = _lib.GNNEA_ADAMW_BLOCK
DESCRIPTOR = len(_lib.AdamwTensor._fields_)  # its 64-bit words
CTL = _lib.GNNEA_ADAMW_CTL_BYTES // 4


def _dense(t):
    """Whether t's elements fill memory without gaps, in whatever order of dimensions."""
    if t.numel() == 0:
        return True
    need = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != need:
            return False
        need *= size
    return True


def _layout(t):
    """(shape, strides) of a dense tensor: which element stands where.  Strides that mean nothing
    (of dimensions of one element, of a tensor of none) are 0."""
    shape = tuple(t.shape)
    if 0 in shape:
        return shape, (0,) * len(shape)
    return shape, tuple(0 if n == 1 else st for n, st in zip(shape, t.stride()))


class AdamW(torch.optim.Optimizer):
    """m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
    p = p (1 - lr weight_decay) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps).

    params          fp32 or bf16 tensors on one HIP device, in any number, or groups of them
    lr              a number, or a one-element fp32 device tensor (read at every step, also by a
                    captured graph)
    state_bits      32, or 8: m in e4m3 and sqrt(v) in 8 bits without a sign, each with one
                    exponent per 256 elements; sqrt(v) is rounded up or down by chance (``seed``),
                    so that small changes are kept on average
    max_norm        scale the gradients of all groups together down to this norm (None: no
                    clipping).  The norm is then in ``grad_norm`` (a device tensor), and a step
                    whose norm is not finite changes nothing; without it, such gradients reach
                    the parameters as in torch.
    A parameter without a gradient is left as it is.  t counts a parameter's own steps, those with a
    gradient, as in torch; parameters of a group with the same history share one counter (and one
    small launch per step).  A captured step goes on with the counters it was captured with: capture
    again after an eager step in which other parameters had gradients.
    Moments keep the order of memory that their parameter had when they were made: a parameter whose
    shape, strides or device is another after that is refused.  A state dict names the order of 8-bit
    codes ("layout"); without it they are taken as row-major."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 state_bits=32, max_norm=None, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("gnnea.AdamW: state_bits must be 8 or 32 (got %r)" % (state_bits,))
        if max_norm is not None and not max_norm > 0:
            raise ValueError("gnnea.AdamW: max_norm must be positive (got %r)" % (max_norm,))
        self.state_bits, self.max_norm = state_bits, max_norm
        self.seed = int(seed) & 0xffffffff
        self.grad_norm = None
        self._order = {}  # the layout that a parameter's moments have
        # of the states that have been compared with their parameter: their tensors, and what the
        # parameter was then (shape, strides, device, length)
        self._known = {}
        self._base = []  # number of a group's first parameter in the hash of the 8-bit rounding
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, group):
        base = sum(len(g["params"]) for g in self.param_groups)
        super().add_param_group(group)
        self._base.append(base)
        try:
            self._check_group(self.param_groups[-1])
        except (TypeError, ValueError):
            self.param_groups.pop()
            self._base.pop()
            raise

    @staticmethod
    def _check_lr(lr):
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32 or not lr.is_cuda:
                raise ValueError("gnnea.AdamW: a tensor lr must be one fp32 value on the device")
        elif not lr >= 0:
            raise ValueError("gnnea.AdamW: lr must not be negative (got %r)" % (lr,))

    @classmethod
    def _check_numbers(cls, group):
        cls._check_lr(group["lr"])
        betas = group["betas"]
        if not group["eps"] > 0 or not group["weight_decay"] >= 0:
            raise ValueError("gnnea.AdamW: eps must be positive and weight_decay not negative")
        if len(betas) != 2 or not 0 <= betas[0] < 1 or not 0 <= betas[1] < 1:
            raise ValueError("gnnea.AdamW: betas must be in [0, 1) (got %r)" % (betas,))

    @classmethod
    def _check_group(cls, group):
        cls._check_numbers(group)
        for name in ("amsgrad", "maximize", "differentiable"):
            if group.get(name):
                raise ValueError("gnnea.AdamW: %s is not done here" % name)
        if group["weight_decay"] and not group.get("decoupled_weight_decay", True):
            raise ValueError("gnnea.AdamW: weight_decay here is decoupled from the gradient")
        if len(set(map(id, group["params"]))) != len(group["params"]):
            raise ValueError("gnnea.AdamW: a parameter is in its group twice")
        for p in group["params"]:
            if p.dtype not in FEATURE_DTYPES:
                raise TypeError("gnnea.AdamW: fp32 or bf16 parameters required (got %s)" % p.dtype)
            if p.is_sparse or not _dense(p):
                raise ValueError("gnnea.AdamW: parameters must be dense and without gaps")

    def __getstate__(self):
        return dict(super().__getstate__(), state_bits=self.state_bits, max_norm=self.max_norm,
                    seed=self.seed, grad_norm=None, _base=self._base,
                    _order=self._order, _known={})

    def _init_state(self, p, step):
        s = self.state[p]
        self._order[p] = _layout(p)
        s["step"] = step
        if self.state_bits == 32:
            s["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            s["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        else:
            n = p.numel()
            s["exp_avg"] = torch.zeros(n, dtype=torch.uint8, device=p.device)
            s["exp_avg_rms"] = torch.zeros(n, dtype=torch.uint8, device=p.device)
            # the exponents of m's and of sqrt(v)'s blocks (any valid one: every code is zero)
            s["scales"] = torch.full((2, -(-n // BLOCK)), 127, dtype=torch.uint8, device=p.device)
        return s

    def _names(self):
        return ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("exp_avg", "exp_avg_rms",
                                                                      "scales")

    def _state_row(self, p, s, shape, stride, device):
        """m, the second moment, the scales and the length of a state, for a descriptor, after p, of
        this shape, strides and device, and its state have been compared."""
        if self.state_bits == 32:
            m, v, scales, at = s["exp_avg"], s["exp_avg_sq"], None, 0
        else:
            m, v, scales = s["exp_avg"], s["exp_avg_rms"], s["scales"]
            at = scales.data_ptr()
        known = self._known.get(id(s))
        if known is not None:
            m0, v0, scales0, shape0, stride0, device0, n = known
            if m is m0 and v is v0 and scales is scales0 and shape == shape0 and \
                    stride == stride0 and device == device0:
                return m.data_ptr(), v.data_ptr(), at, n
        self._check_state(p, s)
        self._known[id(s)] = m, v, scales, shape, stride, device, p.numel()
        return m.data_ptr(), v.data_ptr(), at, p.numel()

    def _check_state(self, p, s):
        order = self._order.setdefault(p, _layout(p))
        if order != _layout(p):
            raise ValueError("gnnea.AdamW: a parameter's shape and strides were %s at its first step "
                             "and are %s now" % (order, _layout(p)))
        n = p.numel()
        for name in self._names():
            t = s[name]
            if t.device != p.device:
                raise ValueError("gnnea.AdamW: a parameter is on %s, its state on %s"
                                 % (p.device, t.device))
            if self.state_bits == 32:
                ok = t.dtype == torch.float32 and _layout(t) == order
            else:
                ok = t.dtype == torch.uint8 and t.is_contiguous() and tuple(t.shape) == (
                    (2, -(-n // BLOCK)) if name == "scales" else (n,))
            if not ok:
                raise ValueError("gnnea.AdamW: a state's %s is not one of its parameter (%s %s)"
                                 % (name, t.dtype, tuple(t.shape)))

    @staticmethod
    def _gradient(p, g, n):
        """g with p's order of elements.  (torch compares the two where a gradient is assigned; the
        parameter's data, type or place may have been replaced since.)"""
        if g.layout is not torch.strided or g.dtype != p.dtype or g.shape != p.shape or \
                g.device != p.device or p.numel() != n:
            raise ValueError("gnnea.AdamW: gradients must be dense and like their parameter")
        if p.is_contiguous():
            return g if g.is_contiguous() else g.contiguous()
        if not _dense(p):
            raise ValueError("gnnea.AdamW: parameters must be dense and without gaps")
        if g.stride() == p.stride():
            return g
        return torch.empty_like(p, memory_format=torch.preserve_format).copy_(g)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # everything is checked before anything is made or launched
        todo, held, device = [], [], None
        state = self.state
        for base, group in zip(self._base, self.param_groups):
            # by counter: the counter, descriptors by type, states without a gradient; under None the
            # parameters (with gradient and index) that take their first step
            counters, c = {}, None
            for i, p in enumerate(group["params"]):
                s, g = state.get(p), p.grad
                if s is not None:
                    step = s["step"]
                    if c is None or c[0] is not step:
                        c = counters.get(id(step))
                        if c is None:
                            c = counters[id(step)] = (step, {}, [])
                    if g is None:
                        c[2].append(s)
                if g is None:
                    continue
                if device is None:
                    _lib.require_device(p)
                    device = p.device
                if p.device != device:
                    raise ValueError("gnnea.AdamW: parameters on more than one device")
                if s is None:
                    c = counters.get(None)
                    if c is None:
                        c = counters[None] = (None, {}, [])
                dtype = p.dtype
                rows = c[1].get(dtype)
                if rows is None:
                    if dtype not in FEATURE_DTYPES:
                        raise TypeError("gnnea.AdamW: fp32 or bf16 parameters required (got %s)"
                                        % dtype)
                    rows = c[1][dtype] = []
                if s is None:
                    g = self._gradient(p, g, p.numel())
                    rows.append((p, g, base + i))
                else:
                    shape, stride = p.shape, p.stride()
                    m, v, scales, n = self._state_row(p, s, shape, stride, device)
                    if g.is_sparse or g.dtype is not dtype or g.shape != shape or \
                            g.stride() != stride or g.device != device:
                        g = self._gradient(p, g, n)
                    rows += (p.data_ptr(), g.data_ptr(), m, v, scales, n, base + i)
                held.append(g)
            counters = [c for c in counters.values() if c[1]]
            if not counters:
                continue
            self._check_numbers(group)  # they may have been replaced since the group was made
            lr = group["lr"]
            if isinstance(lr, torch.Tensor) and lr.device != device:
                raise ValueError("gnnea.AdamW: lr is on %s, the parameters on %s"
                                 % (lr.device, device))
            todo.append((group, counters))
        if any(step is None or idle for _, counters in todo for step, _, idle in counters) and \
                torch.cuda.is_current_stream_capturing():
            raise RuntimeError("gnnea.AdamW: take a step with the same gradients before capturing "
                               "(a captured first step would set the moments to zero, or a counter "
                               "back, at every replay)")
        groups = []
        for group, counters in todo:
            for step, lists, idle in counters:
                if idle:
                    kept = step.clone()
                    for s in idle:
                        s["step"] = kept
                if step is None:
                    step = torch.zeros(1, dtype=torch.int64, device=device)
                    for rows in lists.values():
                        rows[:] = [x for p, g, index in rows for x in (
                            p.data_ptr(), g.data_ptr(),
                            *self._state_row(p, self._init_state(p, step), p.shape, p.stride(),
                                             device), index)]
                arrays = []
                for dtype, rows in lists.items():
                    table = array("q", rows)
                    held.append(table)
                    arrays.append((table.buffer_info()[0], len(table) // DESCRIPTOR, _lib.GNNEA_BF16
                                   if dtype == torch.bfloat16 else _lib.GNNEA_F32))
                groups.append((group, step, arrays))
        if not groups:
            return loss
        L = _lib.lib()
        with _lib.on_device(device):
            stream = stream_of(device)
            n_parts, counts = 0, ()
            if self.max_norm is not None:
                counts = [[int(L.gnnea_adamw_norm_parts(a, c)) for a, c, _ in arrays]
                          for _, _, arrays in groups]
                n_parts = sum(map(sum, counts))
            # the norm's parts (8 bytes each), then the scalars of each update
            scratch = torch.empty(2 * n_parts + len(groups) * CTL, dtype=torch.float32, device=device)
            parts = at = scratch.data_ptr()
            for (_, _, arrays), of in zip(groups, counts):
                for (a, c, code), m in zip(arrays, of):
                    check(L.gnnea_adamw_norm(a, c, code, at, m, stream))
                    at += 8 * m
            for group, step, arrays in groups:
                lr, (b1, b2) = group["lr"], group["betas"]
                on_device = isinstance(lr, torch.Tensor)
                check(L.gnnea_adamw_begin(parts if n_parts else None, n_parts, self.max_norm or 0.0,
                                          b1, b2, 0.0 if on_device else lr,
                                          lr.data_ptr() if on_device else None, self.seed,
                                          step.data_ptr(), at, stream))
                for a, c, code in arrays:
                    check(L.gnnea_adamw_step(a, c, code, self.state_bits, b1, b2, group["eps"],
                                             group["weight_decay"], at, stream))
                at += 4 * CTL
            if self.max_norm is not None:
                self.grad_norm = scratch[2 * n_parts + 4]
        return loss

    @torch.no_grad()
    def moments(self):
        """[(m, second)] of all parameters in order, (None, None) before their first step: with
        32 bits the state's own exp_avg and exp_avg_sq; with 8 bits what the codes of m and of
        sqrt(v) stand for, exactly, in bf16 tensors of the parameter's shape."""
        state, out, rows = self.state, [], []
        for group in self.param_groups:
            for p in group["params"]:
                s = state.get(p)
                if s is None:
                    out.append((None, None))
                elif self.state_bits == 32:
                    out.append((s["exp_avg"], s["exp_avg_sq"]))
                else:
                    row = self._state_row(p, s, p.shape, p.stride(), p.device)
                    m = torch.empty_like(p, dtype=torch.bfloat16)
                    u = torch.empty_like(m)
                    rows += (m.data_ptr(), u.data_ptr(), *row, 0)
                    out.append((m, u))
        if rows:
            device = next(m.device for m, _ in out if m is not None)
            table = array("q", rows)
            with _lib.on_device(device):
                check(_lib.lib().gnnea_adamw_moments(table.buffer_info()[0],
                                                     len(table) // DESCRIPTOR, stream_of(device)))
        return out

    def state_dict(self):
        sd = super().state_dict()
        if self.state_bits == 8:
            state = sd["state"]
            for saved, group in zip(sd["param_groups"], self.param_groups):
                for key, p in zip(saved["params"], group["params"]):
                    if key in state:
                        state[key] = dict(state[key], layout=torch.tensor(
                            self._order.get(p, _layout(p))))
        return sd

    def _loaded_options(self, old, group):
        """The group's options as the saved ones would make them, checked."""
        new = dict(group)
        for k, v in old.items():
            if k == "params":
                continue
            if isinstance(v, torch.Tensor):
                if v.numel() != 1:
                    raise ValueError("gnnea.AdamW: option %s must be one value (got %s)"
                                     % (k, tuple(v.shape)))
                v = float(v)
            new[k] = v
        self._check_group(new)
        return new

    def _loaded_state(self, key, p, got):
        """(step, moments by name) of a saved state, checked against its parameter."""
        if "step" not in got or torch.as_tensor(got["step"]).numel() != 1 or int(got["step"]) < 0:
            raise ValueError("gnnea.AdamW: the state of parameter %s has no step" % (key,))
        n, order = p.numel(), _layout(p)
        if self.state_bits == 32:
            shapes, dtype = dict(exp_avg=p.shape, exp_avg_sq=p.shape), torch.float32
        else:
            shapes = dict(exp_avg=(n,), exp_avg_rms=(n,), scales=(2, -(-n // BLOCK)))
            dtype, was = torch.uint8, got.get("layout")
            if torch.as_tensor(was).tolist() != list(map(list, order)) if was is not None \
                    else not p.is_contiguous():
                raise ValueError("gnnea.AdamW: the codes of parameter %s are in the order %s, the "
                                 "parameter in %s" % (key, "of rows" if was is None else was, order))
        for name, shape in shapes.items():
            t = got.get(name)
            if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != tuple(shape):
                raise ValueError("gnnea.AdamW: %s of parameter %s must be %s %s for state_bits=%d"
                                 % (name, key, tuple(shape), dtype, self.state_bits))
        return int(got["step"]), {name: got[name] for name in shapes}

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Takes the state as it is (codes stay uint8, moments of bf16 parameters stay fp32), all of
        it or, where anything is refused, none."""
        saved = state_dict["param_groups"]
        if len(saved) != len(self.param_groups) or any(
                len(a["params"]) != len(b["params"]) for a, b in zip(saved, self.param_groups)):
            raise ValueError("gnnea.AdamW: the loaded state has other parameter groups")
        plans = []
        for old, group in zip(saved, self.param_groups):
            options = self._loaded_options(old, group)
            states = [(p, self._loaded_state(key, p, state_dict["state"][key]))
                      for key, p in zip(old["params"], group["params"])
                      if state_dict["state"].get(key)]
            plans.append((group, options, states))
        # memory for all of it; what is there is written into: a captured step keeps its addresses
        new = {}
        for group, _, states in plans:
            counter, of, to = {}, {}, {}  # p's counter; a counter's value; a value's counter
            for p, (step, _) in states:
                t = self.state[p]["step"] if p in self.state else None
                if t is not None and t.device == p.device and of.setdefault(id(t), step) == step:
                    counter[p] = t
                    to.setdefault((step, p.device), t)
            for p, (step, moments) in states:
                if p not in counter:
                    if (step, p.device) not in to:
                        to[step, p.device] = torch.zeros(1, dtype=torch.int64, device=p.device)
                    counter[p] = to[step, p.device]
                have = self.state.get(p)
                if have is not None and (self._order.get(p) != _layout(p)
                                         or have["exp_avg"].device != p.device):
                    have = None
                new[p] = s = dict(step=counter[p])
                for name, t in moments.items():
                    s[name] = have[name] if have is not None else \
                        torch.empty_like(p, dtype=t.dtype) if self.state_bits == 32 else \
                        torch.empty(t.shape, dtype=t.dtype, device=p.device)
        for group, options, states in plans:
            for p, (step, moments) in states:
                new[p]["step"].fill_(step)
                for name, t in moments.items():
                    new[p][name].copy_(t)
            lr = group["lr"]
            if isinstance(lr, torch.Tensor):
                options["lr"] = lr if options["lr"] is lr else lr.fill_(options["lr"])
            group.update(options)
        self.state.clear()
        self.state.update(new)
        self._order, self._known = {p: _layout(p) for p in new}, {}
