"""gnnea.optim.AdamW counts each parameter's own steps, as torch's optimizers do."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("max_norm", [None, 1e9])
def test_late_and_intermittent_gradients_against_torch(device, max_norm):
    """Gradients that come first at the eighth step, that stop, that come every third step: the same
    weights as torch.optim.AdamW's.  The gradients are given, so as in a step's own bound each side's
    update is off by 21 u of at most lr / sqrt(1 - b2) each (an update's largest size), and each
    rounds the weight three times a step."""
    from gnnea.optim import AdamW
    g = torch.Generator().manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(n, generator=g).to(device)) for n in (300, 257, 1000, 5)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a = AdamW(ps, lr=1e-2, max_norm=max_norm)
    b = torch.optim.AdamW(qs, lr=1e-2)
    has = (lambda t: True, lambda t: t >= 7, lambda t: t < 4, lambda t: t % 3 == 1)
    for t in range(12):
        for p, q, f in zip(ps, qs, has):
            p.grad = torch.randn(p.shape, generator=g).to(device) if f(t) else None
            q.grad = None if p.grad is None else p.grad.clone()
        a.step()
        b.step()
    for p, q, f in zip(ps, qs, has):
        assert int(a.state[p]["step"]) == int(b.state[q]["step"]) == sum(map(f, range(12)))
        tol = 2 * 12 * (21 * U * 1e-2 / 0.001 ** 0.5 + 3 * U * q.detach().abs())
        assert bool(((p - q).detach().abs() <= tol).all())


def test_a_state_of_torchs_goes_on(device):
    """Steps of torch's AdamW, its state loaded, more steps: as torch's, where the parameters' steps
    differ."""
    from gnnea.optim import AdamW
    g = torch.Generator().manual_seed(1)
    qs = [torch.nn.Parameter(torch.randn(64, generator=g).to(device)) for _ in range(2)]
    b = torch.optim.AdamW(qs, lr=1e-2)
    grads = [[torch.randn(64, generator=g).to(device) for _ in qs] for _ in range(9)]
    ps = a = None
    for t in range(9):
        if t == 5:
            ps = [torch.nn.Parameter(q.detach().clone()) for q in qs]
            a = AdamW(ps, lr=1.0)
            a.load_state_dict(b.state_dict())
        for opt, xs in ((b, qs), (a, ps)):
            if opt is None:
                continue
            for x, gr, late in zip(xs, grads[t], (False, True)):
                x.grad = None if late and t < 3 else gr.clone()
            opt.step()
    for p, q, n in zip(ps, qs, (9, 6)):
        assert int(a.state[p]["step"]) == n
        tol = 2 * 9 * (21 * U * 1e-2 / 0.001 ** 0.5 + 3 * U * q.detach().abs())
        assert bool(((p - q).detach().abs() <= tol).all())


def test_a_captured_step_after_a_late_gradient(device):
    """Two counters in one captured step: both go on at every replay."""
    from gnnea.optim import AdamW

    def make():
        ps = [torch.nn.Parameter(torch.ones(100, device=device)) for _ in range(2)]
        opt = AdamW(ps, lr=1e-2)
        for t in range(3):
            for i, p in enumerate(ps):
                p.grad = torch.full_like(p, 0.5 + t) if i == 0 or t == 2 else None
            opt.step()
        return ps, opt
    (ps, one), (qs, two) = make(), make()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.step()
    for t in range(4):
        for p, q in zip(ps, qs):
            p.grad.fill_(0.1 * t - 0.2)
            q.grad.fill_(0.1 * t - 0.2)
        graph.replay()
        two.step()
        torch.cuda.synchronize()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q) and torch.equal(one.state[p]["step"], two.state[q]["step"])
    assert [int(one.state[p]["step"]) for p in ps] == [7, 5]
