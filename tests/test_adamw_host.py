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
