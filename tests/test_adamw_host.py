"""gnnea.optim.AdamW's host side without a device: what reaches the library's calls, and what is
refused before them.  The library is replaced by a record of its calls; nothing is computed."""
import contextlib

import pytest
import torch


class Calls:
    """Stands for libgnnea.so: keeps the names of the calls, returns 0."""

    def __init__(self):
        self.names = []

    def __getattr__(self, name):
        def call(*args):
            self.names.append(name)
            return 0
        return call

    def count(self, name):
        return self.names.count(name)


@pytest.fixture
def lib(monkeypatch):
    from gnnea import _lib, optim
    calls = Calls()
    monkeypatch.setattr(_lib, "lib", lambda: calls)
    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    monkeypatch.setattr(_lib, "on_device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(optim, "stream_of", lambda d: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return calls


def parameters(*shapes, dtype=torch.float32):
    ps = [torch.nn.Parameter(torch.zeros(s, dtype=dtype)) for s in shapes]
    for p in ps:
        p.grad = torch.ones_like(p)
    return ps


def refused(lib, opt, error=ValueError):
    """A step raises, and raises before the first call."""
    before = len(lib.names)
    with pytest.raises(error):
        opt.step()
    assert len(lib.names) == before


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("first", [True, False])
def test_a_type_that_changed(lib, bits, dtype, first):
    """model.half() or model.double() after the optimizer was made: elements of 2 or 8 bytes would be
    read and written as 4."""
    from gnnea.optim import AdamW
    p, q = parameters((8,), (4, 6))
    opt = AdamW([p, q], state_bits=bits)
    if not first:
        opt.step()
        assert lib.count("gnnea_adamw_step") == 1
    q.data = q.data.to(dtype)
    q.grad = torch.ones_like(q)
    refused(lib, opt, TypeError)
    q.data = q.data.bfloat16()  # fp32 or bf16: both are known, the moments stay
    q.grad = torch.ones_like(q)
    opt.step()


def test_gradients_that_are_not_the_parameters(lib):
    """A gradient left behind by a replaced parameter: another place, another shape."""
    from gnnea.optim import AdamW
    p, = parameters((4, 6))
    with pytest.raises(ValueError):
        AdamW._gradient(p, torch.ones(4, 6, device="meta"), 24)
    opt = AdamW([p])
    p.data = torch.zeros(6, 4)
    assert p.grad.shape == (4, 6)
    refused(lib, opt)


def transposed(t):
    return t.t().contiguous().t()


@pytest.mark.parametrize("bits", [32, 8])
def test_an_order_that_changed(lib, bits):
    """Moments belong to elements by the order of memory: a parameter of another order, or of
    another shape of as many elements, is refused by step and by moments()."""
    from gnnea.optim import AdamW
    for new in (transposed(torch.ones(4, 6)), torch.ones(6, 4), torch.ones(24)):
        p, q = parameters((3,), (4, 6))
        opt = AdamW([p, q], state_bits=bits)
        opt.step()
        was = q.data
        q.data, q.grad = new, torch.ones_like(new)
        refused(lib, opt)
        if bits == 8:
            with pytest.raises(ValueError):
                opt.moments()
            assert not lib.count("gnnea_adamw_moments")
        q.data, q.grad = was, torch.ones_like(was)
        opt.step()
    p, = parameters((1, 5))  # one row: its stride means nothing
    opt = AdamW([p], state_bits=bits)
    opt.step()
    p.data = torch.zeros(5, 1).t()
    p.grad = torch.ones(1, 5)
    opt.step()


def test_codes_are_saved_with_their_order(lib):
    """8-bit codes lie flat in memory order, so a state dict names it: into a parameter of another
    order they are refused; without a name they are row-major."""
    import copy
    from gnnea.optim import AdamW
    row, = parameters((4, 6))
    col = torch.nn.Parameter(transposed(torch.zeros(4, 6)))
    col.grad = torch.ones_like(col)
    one, two = AdamW([row], state_bits=8), AdamW([col], state_bits=8)
    one.step()
    two.step()
    a, b = one.state_dict(), two.state_dict()
    assert "layout" not in one.state[row]
    for opt, other in ((one, b), (two, a)):
        with pytest.raises(ValueError):
            opt.load_state_dict(other)
    one.load_state_dict(copy.deepcopy(a))
    two.load_state_dict(copy.deepcopy(b))
    for sd in (a, b):
        sd["state"][0].pop("layout")
    one.load_state_dict(a)
    with pytest.raises(ValueError):
        two.load_state_dict(b)
    copy.deepcopy(one).step()
    with pytest.raises(ValueError):  # (the codes' own order, not the one that the parameter has now)
        row.data = transposed(row.data)
        AdamW([row], state_bits=8).load_state_dict(one.state_dict())


def test_32_bit_moments_follow_their_elements(lib):
    """32-bit moments have their parameter's shape: loaded into another order, each goes to its own
    element, also where the parameter's order changed after its first step."""
    from gnnea.optim import AdamW
    p, = parameters((4, 6))
    opt = AdamW([p])
    opt.step()
    m = torch.arange(24.0).view(4, 6)
    opt.state[p]["exp_avg"].copy_(m)
    sd = opt.state_dict()
    p.data, p.grad = transposed(p.data), None
    opt.load_state_dict(sd)
    s = opt.state[p]
    assert torch.equal(s["exp_avg"], m) and s["exp_avg"].stride() == p.stride()
    p.grad = torch.ones_like(p)
    opt.step()


def snapshot(opt):
    import copy
    state = {p: {k: (v, v.clone()) for k, v in s.items()} for p, s in opt.state.items()}
    groups = [{k: copy.deepcopy(v) for k, v in g.items() if k != "params"} for g in opt.param_groups]
    return state, groups, dict(opt._order)


def assert_unchanged(opt, was):
    state, groups, order = was
    assert set(opt.state) == set(state) and opt._order == order
    for p, s in state.items():
        assert set(opt.state[p]) == set(s)
        for k, (same, value) in s.items():
            assert opt.state[p][k] is same and torch.equal(same, value), k
    for g, old in zip(opt.param_groups, groups):
        assert {k: v for k, v in g.items() if k != "params"} == old


def spoil(sd, how):
    second, group = sd["state"][1], sd["param_groups"][1]
    if how == "shape":
        second["exp_avg"] = second["exp_avg"].reshape(-1)[:-1]
    elif how == "type":
        second["exp_avg"] = second["exp_avg"].double()
    elif how == "name":
        del second["exp_avg"]
    elif how == "step":
        del second["step"]
    elif how == "steps":
        second["step"] = torch.zeros(2)
    elif how == "negative":
        second["step"] = -1
    elif how == "group":
        sd["param_groups"].pop()
    elif how == "betas":
        group["betas"] = (0.9, 1.0)
    elif how == "lr":
        group["lr"] = -1.0
    elif how == "lrs":
        group["lr"] = torch.ones(2)
    elif how == "eps":
        group["eps"] = 0.0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["shape", "type", "name", "step", "steps", "negative", "group",
                                 "betas", "lr", "lrs", "eps", "bits"])
def test_a_refused_load_changes_nothing(lib, bits, how):
    """The first parameter's part of the dict is sound, and not taken: nor its step or options."""
    import copy
    from gnnea.optim import AdamW

    def make(bits, lr):
        ps = parameters((5,), (4, 6))
        opt = AdamW([dict(params=[ps[0]]), dict(params=[ps[1]], lr=lr)], lr=lr, state_bits=bits)
        opt.step()
        for p in ps:
            opt.state[p]["step"].fill_(round(lr * 1000))
            opt.state[p]["exp_avg"].fill_(3)
        return opt
    live, other = make(bits, 0.005), make(8 if (how == "bits") == (bits == 32) else 32, 0.099)
    sd = copy.deepcopy(other.state_dict())
    spoil(sd, how)
    was = snapshot(live)
    with pytest.raises((ValueError, TypeError)):
        live.load_state_dict(sd)
    assert_unchanged(live, was)
    live.step()
    live.load_state_dict(make(bits, 0.099).state_dict())
    assert int(live.state[live.param_groups[0]["params"][0]]["step"]) == 99
    assert live.param_groups[1]["lr"] == 0.099


@pytest.mark.parametrize("option,ok", [
    (dict(maximize=True), False), (dict(amsgrad=True), False), (dict(differentiable=True), False),
    (dict(decoupled_weight_decay=False, weight_decay=0.1), False),
    (dict(decoupled_weight_decay=False, weight_decay=0.0), True),
    (dict(maximize=False, amsgrad=False, foreach=True, initial_lr=0.1), True)])
def test_options_that_the_step_does_not_do(lib, option, ok):
    """torch's optimizers' options that would change the update are refused where they are on: in a
    group, and in a state dict of torch's."""
    from gnnea.optim import AdamW
    p, = parameters((3,))
    opt = AdamW([p])
    sd = opt.state_dict()
    sd["param_groups"][0].update(option)
    if ok:
        opt.load_state_dict(sd)
        AdamW([dict(params=[p], **option)]).step()
        return
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)
    assert not set(option) - {"weight_decay"} & set(opt.param_groups[0])
    with pytest.raises(ValueError):
        AdamW([dict(params=[p], **option)])


def test_a_state_of_torchs(lib):
    """torch.optim.Adam's and AdamW's own dicts, as they are by default."""
    from gnnea.optim import AdamW
    p, = parameters((3,))
    for other in (torch.optim.Adam([p]), torch.optim.AdamW([p])):
        other.step()
        opt = AdamW([p])
        opt.load_state_dict(other.state_dict())
        assert torch.equal(opt.state[p]["exp_avg"], other.state[p]["exp_avg"])
        assert int(opt.state[p]["step"]) == 1
    with pytest.raises(ValueError):
        AdamW([p]).load_state_dict(torch.optim.Adam([p], weight_decay=0.1).state_dict())


def counters(opt, ps):
    return [opt.state[p]["step"].data_ptr() for p in ps]


def test_a_counter_for_each_history(lib, monkeypatch):
    """t is a parameter's own: those whose gradients came in the same steps share a counter (one
    launch before the updates), a parameter that comes later or stays out has its own from there."""
    from gnnea.optim import AdamW
    ps = parameters((3,), (4,), (5,), (6,))
    ps[3].grad = None
    opt = AdamW(ps)
    opt.step()
    assert len(set(counters(opt, ps[:3]))) == 1 and lib.count("gnnea_adamw_begin") == 1
    first = counters(opt, ps[:1])[0]
    ps[3].grad = torch.ones(6)
    opt.step()  # the newcomer counts from 0
    assert counters(opt, ps[:3]) == [first] * 3 and counters(opt, ps)[3] != first
    assert lib.count("gnnea_adamw_begin") == 1 + 2
    ps[1].grad = None
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    before = len(lib.names)
    with pytest.raises(RuntimeError):  # a graph would set the counter back at every replay
        opt.step()
    assert len(lib.names) == before and counters(opt, ps[:3]) == [first] * 3
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    opt.state[ps[0]]["step"].fill_(7)
    opt.step()  # the one that stays out keeps the old count, in a counter of its own
    assert counters(opt, [ps[0], ps[2]]) == [first] * 2 and counters(opt, ps)[1] != first
    assert int(opt.state[ps[1]]["step"]) == 7
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    opt.step()  # the same parameters as in the step before: nothing to part


def test_steps_that_differ_are_loaded(lib):
    """A state whose parameters have taken different numbers of steps keeps each; counters that are
    there are written into."""
    from gnnea.optim import AdamW
    ps = parameters((3,), (4,), (5,))
    other = torch.optim.AdamW(ps)
    other.step()
    sd = other.state_dict()
    for i, t in enumerate((1000, 1, 1000)):
        sd["state"][i]["step"] = torch.tensor(float(t))
    opt = AdamW(ps)
    opt.load_state_dict(sd)
    assert [int(opt.state[p]["step"]) for p in ps] == [1000, 1, 1000]
    assert len(set(counters(opt, ps))) == 2
    was = counters(opt, ps)
    sd["state"][1]["step"] = torch.tensor(5.0)
    opt.load_state_dict(sd)
    assert counters(opt, ps) == was and [int(opt.state[p]["step"]) for p in ps] == [1000, 5, 1000]
    sd["state"][2]["step"] = torch.tensor(2.0)
    opt.load_state_dict(sd)
    assert [int(opt.state[p]["step"]) for p in ps] == [1000, 5, 2]
    opt.load_state_dict(opt.state_dict())
    assert [int(opt.state[p]["step"]) for p in ps] == [1000, 5, 2]
    lib.names.clear()
    opt.step()
    assert lib.count("gnnea_adamw_begin") == 3


def test_a_refused_step_leaves_no_state(lib):
    """A later group's refusal comes before anything is made or parted for an earlier one."""
    from gnnea.optim import AdamW
    p, q, r = parameters((3,), (4,), (5,))
    opt = AdamW([dict(params=[p, q]), dict(params=[r])])
    r.data = torch.zeros(5).double()
    refused(lib, opt, TypeError)
    assert not opt.state


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shape", [(0,), (0, 4), (5, 0), (2, 0, 3)])
def test_parameters_without_elements(lib, shape, bits):
    """Dense whatever their strides; a step, its state and loading it leave the others theirs."""
    from gnnea.optim import AdamW
    p, q = parameters(shape, (3,))
    opt = AdamW([p, q], state_bits=bits)
    opt.step()
    opt.load_state_dict(opt.state_dict())
    opt.step()
    assert opt.state[p]["exp_avg"].numel() == 0 and lib.count("gnnea_adamw_step") == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_was_replaced(lib, bits):
    """Tensors put into the state by hand are held to its parameter's size, type, order and place."""
    from gnnea.optim import AdamW
    p, = parameters((40, 30))
    opt = AdamW([p], state_bits=bits)
    opt.step()
    s = opt.state[p]
    for name in opt._names():
        was = s[name]
        bad = [was.double(), was.flatten()[:-1], was.to("meta")]
        bad += [transposed(was)] if was.dim() == 2 and was.shape[0] > 1 else []
        for t in bad:
            s[name] = t
            refused(lib, opt)
        s[name] = was.clone()
        opt.step()


@pytest.mark.parametrize("name,value", [("betas", (0.9, 1.0)), ("betas", (-0.1, 0.9)), ("eps", 0.0),
                                        ("weight_decay", -1.0), ("eps", float("nan"))])
def test_numbers_that_were_replaced(lib, name, value):
    """Set after the group was made: refused before the first group's update."""
    from gnnea.optim import AdamW
    p, q = parameters((3,), (4,))
    opt = AdamW([dict(params=[p]), dict(params=[q])], max_norm=1.0)
    opt.step()
    opt.param_groups[1][name] = value
    refused(lib, opt)
