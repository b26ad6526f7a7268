"""gnnea.optim.AdamW without clipping, where a gradient is not finite: as in torch, that element is
lost and no other, also with 8-bit moments, whose blocks of 256 share their exponents."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("first", [True, False])
def test_one_element_is_lost(device, bits, bad, dtype, first):
    """Bit for bit: every other element, its moments included, is what it is where that gradient is
    0 instead, in this step and in the ones after it (3e38: its square is not finite.  With 32 bits
    its second moment is infinite from then on and its update 0; with 8 bits it is lost)."""
    from gnnea.optim import AdamW
    n, at = 700, 300
    g = torch.Generator().manual_seed(0)
    start = torch.randn(n, generator=g).to(dtype).to(device)
    p, q = (torch.nn.Parameter(start.clone()) for _ in range(2))
    one, two = (AdamW([x], lr=1e-2, state_bits=bits, seed=5) for x in (p, q))
    rest = torch.ones(n, dtype=torch.bool, device=device)
    rest[at] = False
    for t in range(5):
        gr = torch.randn(n, generator=g).to(dtype).to(device)
        gr[at] = 0
        q.grad = gr
        p.grad = gr.clone()
        if t == (0 if first else 2):
            p.grad[at] = bad
        one.step()
        two.step()
        for (a, b) in ((p, q),) + tuple(zip(one.moments()[0], two.moments()[0])):
            assert torch.equal(a.detach()[rest], b.detach()[rest]), t
    if bits == 8 or not math.isfinite(bad):
        assert not bool(torch.isfinite(p[at]))
    assert bool(torch.isfinite(p[rest]).all())


def test_a_block_that_is_lost_whole(device):
    """All of a block's gradients NaN: the block is lost, its neighbours are not, nothing hangs on
    the exponents of a block without a finite value."""
    from gnnea.optim import AdamW
    p = torch.nn.Parameter(torch.ones(1000, device=device))
    opt = AdamW([p], state_bits=8)
    for _ in range(3):
        p.grad = torch.ones_like(p)
        p.grad[256:512] = math.nan
        opt.step()
    lost = torch.isnan(p.detach())
    assert bool(lost[256:512].all()) and int(lost.sum()) == 256
