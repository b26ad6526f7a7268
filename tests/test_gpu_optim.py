"""gnnea.optim.AdamW: the update against fp64, the 8-bit codes bit for bit against a numpy
restatement, clipping, state dicts, captured steps.

Tolerances (u = 2^-24).  The clipped gradient is off by 2 u (its factor, the product).
    m    b1's term: the constant, the product, the sum, 3 u; g's: 2 + 3 = 5 u
    v    b2's term 3 u; g's: squared 2 * 2 + 1, the constant, the product, the sum, 8 u
    p    m 5, 1 / (1 - b1^t) 1, lr 1, their products 2; the root (8 / 2 + 1), its factor and product 2,
         eps 1, the reciprocal 2 (one last place), its product 1, the product with lr 1: 21 u of the update, 3 u of p (decay, product,
         difference) and eps / 2 of the value for its type
Codes: every operation of the restatement rounds as the kernel's does
(fp32 products and sums of the second moment, fp64 for the first), so they are equal.
"""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
B1, B2 = 0.9, 0.999
M32 = np.uint32


def mix(h):
    h = (h ^ (h >> M32(16))) * M32(0x85ebca6b)
    h = (h ^ (h >> M32(13))) * M32(0xc2b2ae35)
    return h ^ (h >> M32(16))


def e4m3(code):
    return torch.from_numpy(code.copy()).view(torch.float8_e4m3fn).float().numpy()


def decode_u(code):
    v = ((code.astype(np.uint32) << M32(19)) + M32(112 << 23)).view(np.float32)
    return np.where(code == 0, np.float32(0), v)


def codes(mc, uc, sc, g, t, index, seed):
    """One step of the moments in numpy: new codes, scales and fp32 moments."""
    n = g.size
    nb = -(-n // 256)
    blk = np.arange(n) // 256
    p2 = lambda e: (e.astype(np.uint32) << M32(23)).view(np.float32)  # noqa: E731
    m = e4m3(mc) * p2(sc[0])[blk]
    u = decode_u(uc) * p2(sc[1])[blk]
    m = (m.astype(np.float64) * B1 + g.astype(np.float64) * (1 - B1)).astype(np.float32)
    u = np.sqrt(u * u * np.float32(B2) + g * g * np.float32(1 - B2))
    new = np.zeros((2, nb), np.uint8)
    for b in range(nb):
        at = slice(b * 256, min(n, b * 256 + 256))
        top = np.abs(m[at]).max().view(np.uint32)
        new[0, b] = max(1, int((int(top) + (1 << 21)) >> 23) - 8)
        new[1, b] = min(254, max(17, (int(u[at].max().view(np.uint32)) + (1 << 19)) >> 23))
    mq = torch.from_numpy(m / p2(new[0])[blk]).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    with np.errstate(over="ignore"):
        key = mix(M32((seed + 0x9e3779b9 * t) & 0xffffffff) + M32((0x85ebca6b * index) & 0xffffffff))
        chance = mix(np.arange(n, dtype=np.uint32) + key) >> M32(13)
    bits = (u / p2(new[1])[blk]).view(np.uint32).astype(np.int64) - (112 << 23) + chance
    uq = np.where(u == 0, 0, np.clip(bits >> 19, 1, 255)).astype(np.uint8)
    return mq, uq, new, m, u


def make(device, shapes, dtype, seed=0, std=0.01):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).to(device)) for s in shapes]

    def grads(k):
        gg = torch.Generator().manual_seed(1000 + k)
        for p in ps:
            p.grad = (torch.randn(p.shape, generator=gg) * std).to(dtype).to(device)
    return ps, grads


SHAPES = [(1,), (3, 5), (256,), (255, 1), (257,), (300, 300), (300,), (1025, 7), (4099,), (0, 4)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_norm", [None, 0.05, 1e6])
def test_32_bits_against_fp64(device, dtype, max_norm):
    from gnnea.optim import AdamW
    ps, grads = make(device, SHAPES, dtype)
    opt = AdamW(ps, lr=3e-3, betas=(B1, B2), eps=1e-8, weight_decay=0.1, max_norm=max_norm)
    m64 = [torch.zeros(p.shape).double() for p in ps]
    v64 = [torch.zeros(p.shape).double() for p in ps]
    for t in range(1, 5):
        grads(t)
        before = [p.detach().double().cpu() for p in ps]
        g = [p.grad.double().cpu() for p in ps]
        old = [(m.clone(), v.clone()) for m, v in zip(m64, v64)]
        opt.step()
        norm = float(torch.sqrt(sum((x ** 2).sum() for x in g)))
        by = 1.0 if max_norm is None else min(1.0, max_norm / (norm + 1e-6))
        if max_norm is not None:
            assert abs(float(opt.grad_norm) - norm) <= 4 * U * norm
        for i, (p, (m, v)) in enumerate(zip(ps, opt.moments())):
            gi = g[i] * by
            m64[i] = B1 * old[i][0] + (1 - B1) * gi
            v64[i] = B2 * old[i][1] + (1 - B2) * gi ** 2
            em = (m.double().cpu() - m64[i]).abs()
            ev = (v.double().cpu() - v64[i]).abs()
            assert bool((em <= 5 * U * ((B1 * old[i][0]).abs() + 0.1 * gi.abs()) + 1e-38).all())
            assert bool((ev <= 8 * U * v64[i] + 1e-38).all())
            up = 3e-3 * (m64[i] / (1 - B1 ** t)) / ((v64[i] / (1 - B2 ** t)).sqrt() + 1e-8)
            want = before[i] * (1 - 3e-4) - up
            ma = 3e-3 * (((B1 * old[i][0]).abs() + 0.1 * gi.abs()) / (1 - B1 ** t)) / (
                (v64[i] / (1 - B2 ** t)).sqrt() + 1e-8)
            tol = 3 * U * before[i].abs() + 21 * U * ma + torch.finfo(dtype).eps / 2 * want.abs()
            assert bool(((p.detach().double().cpu() - want).abs() <= tol + 1e-38).all()), (t, i)
            # what the next step starts from
            m64[i], v64[i] = m.double().cpu(), v.double().cpu()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_8_bit_codes(device, dtype):
    """Codes, scales and values equal to the restatement over several steps, gradients of wide
    range and zeros among them; the update uses the moments before rounding."""
    from gnnea.optim import AdamW
    ps, grads = make(device, SHAPES, dtype, 2)
    opt = AdamW(ps, lr=3e-3, betas=(B1, B2), weight_decay=0.1, state_bits=8, seed=77)
    have = [(np.zeros(p.numel(), np.uint8), np.zeros(p.numel(), np.uint8),
             np.full((2, -(-p.numel() // 256)), 127, np.uint8)) for p in ps]
    for t in range(1, 6):
        grads(t)
        for p in ps:  # from 1e-9 to 10 within one block, every seventh zero
            f = torch.logspace(-9, 1, 97).to(device).repeat(p.numel() // 97 + 1)[:p.numel()]
            f[::7] = 0
            p.grad = (p.grad.float() * f.view(p.shape)).to(dtype)
        before = [p.detach().double().cpu() for p in ps]
        opt.step()
        for i, (p, (mv, uv)) in enumerate(zip(ps, opt.moments())):
            if not p.numel():
                continue
            mq, uq, sc, m, u = codes(*have[i], p.grad.float().cpu().numpy().reshape(-1), t, i, 77)
            s = opt.state[p]
            assert np.array_equal(s["scales"].cpu().numpy(), sc), (t, i)
            assert np.array_equal(s["exp_avg"].cpu().numpy() & 0x7f, mq & 0x7f), (t, i)
            assert np.array_equal(s["exp_avg"].cpu().numpy()[mq & 0x7f != 0], mq[mq & 0x7f != 0])
            assert np.array_equal(s["exp_avg_rms"].cpu().numpy(), uq), (t, i)
            blk = np.arange(p.numel()) // 256
            p2 = np.exp2(sc.astype(np.float64) - 127)
            assert np.array_equal(mv.double().cpu().numpy().reshape(-1),
                                  e4m3(mq).astype(np.float64) * p2[0][blk])
            assert np.array_equal(uv.double().cpu().numpy().reshape(-1),
                                  decode_u(uq).astype(np.float64) * p2[1][blk])
            up = 3e-3 * (m.astype(np.float64) / (1 - B1 ** t)) / (
                u.astype(np.float64) / np.sqrt(1 - B2 ** t) + 1e-8)
            b = before[i].numpy().reshape(-1)
            want = b * (1 - 3e-4) - up
            tol = 3 * U * np.abs(b) + 21 * U * np.abs(up) + torch.finfo(dtype).eps / 2 * np.abs(want)
            got = p.detach().double().cpu().numpy().reshape(-1)
            assert (np.abs(got - want) <= tol + 1e-38).all(), (t, i)
            have[i] = (mq, uq, sc)


def test_8_bits_keep_the_mean(device):
    """A constant gradient after another: sqrt(v) follows by chance what nearest rounding would
    never move.  65536 elements that start at v = 1 under g = 2: after 50 steps v = 4 - 3 0.999^50,
    u = 1.0683; each of 50 roundings errs by at most a step of 1/16, with mean 0, so the mean over
    65536 elements is off by at most 6 * sqrt(50) / 16 / 2 / 256 = 0.0052 (six deviations, each at
    most half a step) and, the root of a mean being above the mean of roots, by var / 2u = 0.0015."""
    from gnnea.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(65536, device=device))
    opt = AdamW([p], lr=0.0, betas=(B1, B2), state_bits=8)
    p.grad = torch.full_like(p, 1.0)
    opt.step()
    s = opt.state[p]
    s["exp_avg_rms"].fill_(15 * 16)  # 1.0 under the exponent 127
    s["scales"].fill_(127)
    p.grad.fill_(2.0)
    for _ in range(50):
        opt.step()
    u = opt.moments()[0][1].float()
    assert abs(float(u.mean()) - (4 - 3 * 0.999 ** 50) ** 0.5) < 0.0067
    assert int(u.unique().numel()) > 1


def test_norm_that_is_not_finite(device):
    """With max_norm the whole step is left out, without it NaN reaches the parameter."""
    from gnnea.optim import AdamW
    for bits in (32, 8):
        ps, grads = make(device, [(300,), (300, 3)], torch.float32)
        opt = AdamW(ps, state_bits=bits, max_norm=1.0)
        grads(1)
        opt.step()
        want = [p.detach().clone() for p in ps]
        st = [{k: v.clone() for k, v in opt.state[p].items()} for p in ps]
        for bad in (float("nan"), float("inf")):
            ps[1].grad[7, 1] = bad
            opt.step()
            for p, w, s in zip(ps, want, st):
                assert torch.equal(p.detach(), w)
                for k, v in s.items():
                    assert torch.equal(opt.state[p][k], v), k
        free = AdamW([ps[1]], state_bits=bits)
        free.step()
        assert not bool(torch.isfinite(ps[1]).all())


def test_many_tensors_groups_and_missing_gradients(device):
    """200 tensors (several launches), two groups of different rates, some without a gradient:
    equal, bit for bit, to one optimizer per tensor with the same numbers."""
    from gnnea.optim import AdamW
    shapes = [((i * 37) % 501 + 1,) for i in range(200)]
    ps, grads = make(device, shapes, torch.float32, 3)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = AdamW([dict(params=ps[:120], lr=1e-2), dict(params=ps[120:], lr=1e-3, weight_decay=0.0)])
    each = [AdamW([q], lr=1e-2 if i < 120 else 1e-3, weight_decay=1e-2 if i < 120 else 0.0)
            for i, q in enumerate(qs)]
    for t in range(3):
        grads(t)
        for i, (p, q) in enumerate(zip(ps, qs)):
            if i % 11 == 5:
                p.grad = None
            q.grad = p.grad
        opt.step()
        for o in each:
            o.step()
    for i, (p, q) in enumerate(zip(ps, qs)):
        assert torch.equal(p, q), i
    assert opt.moments()[5] == (None, None)


def test_strides_alignment_streams(device):
    """Parameters in column-major order, views at odd offsets, gradients in another order."""
    from gnnea.optim import AdamW
    for bits in (32, 8):
        buf = torch.randn(5000, device=device)
        a = torch.nn.Parameter(buf[1:1 + 900].view(30, 30))
        b = torch.nn.Parameter(buf[1001:1001 + 700].view(70, 10).t())
        ga, gb = torch.randn(30, 30, device=device), torch.randn(10, 70, device=device)
        c, d = (torch.nn.Parameter(t.detach().clone().contiguous()) for t in (a, b.t()))
        rest = buf.clone()
        a.grad, b.grad = ga.t().contiguous().t(), gb
        c.grad, d.grad = ga, gb.t().contiguous()
        one, two = AdamW([a, b], state_bits=bits), AdamW([c, d], state_bits=bits)
        s = torch.cuda.Stream(device)
        s.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(s):
            one.step()
        torch.cuda.current_stream(device).wait_stream(s)
        two.step()
        assert torch.equal(a, c) and torch.equal(b.t(), d)
        keep = torch.ones(5000, dtype=torch.bool)
        keep[1:901] = keep[1001:1701] = False
        assert torch.equal(buf.detach().cpu()[keep], rest.cpu()[keep])


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_and_capture(device, bits):
    """A run that is saved, loaded and gone on with, one that is not, and one whose steps are
    replays of a captured graph (a scheduler changing the rate): the same bits."""
    from gnnea.optim import AdamW
    shapes = [(300, 300), (300,), (77,)]

    def fresh():
        ps, grads = make(device, shapes, torch.float32, 5)
        grads(0)
        lr = torch.full((1,), 1e-2, device=device)
        return ps, grads, lr, AdamW(ps, lr=lr, state_bits=bits, max_norm=0.5, seed=3)

    def set_grads(ps, k):
        gg = torch.Generator().manual_seed(50 + k)
        for p in ps:
            p.grad.copy_(torch.randn(p.shape, generator=gg))

    def go(n):
        ps, grads, lr, opt = fresh()
        for k in range(n):
            set_grads(ps, k)
            lr.fill_(1e-2 / (k + 1))
            opt.step()
        return ps, lr, opt
    want, _, wopt = go(6)
    ps, lr, opt = go(3)
    sd = copy.deepcopy(opt.state_dict())
    assert all(s["exp_avg"].dtype == (torch.uint8 if bits == 8 else torch.float32)
               for s in sd["state"].values())
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    opt2 = AdamW(qs, lr=1.0, state_bits=bits, max_norm=0.5, seed=3)
    opt2.load_state_dict(sd)
    for k in range(3, 6):
        set_grads(qs, k)
        opt2.param_groups[0]["lr"] = 1e-2 / (k + 1)
        opt2.step()
    for a, b in zip(want, qs):
        assert torch.equal(a, b)
    ps, grads, lr, opt = fresh()
    set_grads(ps, 0)
    opt.step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    for k in range(1, 6):
        set_grads(ps, k)
        lr.fill_(1e-2 / (k + 1))
        g.replay()
        torch.cuda.synchronize()
    for a, b in zip(want, ps):
        assert torch.equal(a, b)
    for (m, u), (m2, u2) in zip(wopt.moments(), opt.moments()):
        assert torch.equal(m, m2) and torch.equal(u, u2)


def test_refusals(device):
    from gnnea.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4, 4, device=device))
    for kw in (dict(lr=-1.0), dict(eps=0.0), dict(betas=(1.0, 0.9)), dict(weight_decay=-1.0),
               dict(state_bits=16), dict(max_norm=0.0), dict(lr=torch.ones(2, device=device))):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(TypeError):
        AdamW([torch.nn.Parameter(torch.zeros(4, device=device).half())])
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(4, 8, device=device)[:, :4])])
    opt = AdamW([p])
    p.grad = torch.zeros(4, 4, device=device).to_sparse()
    with pytest.raises(ValueError):
        opt.step()
    p.grad = torch.zeros(4, 4, device=device)
    opt.step()
    with pytest.raises(ValueError):
        AdamW([p], state_bits=8).load_state_dict(opt.state_dict())
    q = torch.nn.Parameter(torch.zeros(4, device=device))
    q.grad = torch.zeros(4, device=device)
    g = torch.cuda.CUDAGraph()
    first = AdamW([q])
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(g):
            first.step()


def test_offsets_past_32_bits(device):
    """A bf16 tensor of 2^32 + 4097 elements, all alike: all alike after a step, and as a small
    tensor's."""
    from gnnea.optim import AdamW
    got = []
    for n in (2 ** 32 + 4097, 5):
        p = torch.nn.Parameter(torch.full((n,), 1.5, dtype=torch.bfloat16, device=device))
        p.grad = torch.full_like(p, 0.25)
        opt = AdamW([p], lr=0.1, max_norm=None)
        opt.step()
        m, v = opt.moments()[0]
        for t in (p.detach(), m, v):
            lo, hi = torch.aminmax(t)
            assert lo == hi
        got.append((p.detach()[-1].item(), m[-1].item(), v[-1].item()))
        del p, opt, m, v, t
        torch.cuda.empty_cache()
    assert got[0] == got[1]


def test_copies_duplicates_and_rates(device):
    """A deep copy goes on by itself; the same parameter twice, and a rate on the host, are refused;
    loading writes into the state that is there."""
    from gnnea.optim import AdamW
    p = torch.nn.Parameter(torch.ones(300, device=device))
    with pytest.raises(ValueError):
        AdamW([p, p])
    with pytest.raises(ValueError):
        AdamW([p], lr=torch.ones(1))
    p.grad = torch.full_like(p, 0.5)
    opt = AdamW([p], state_bits=8, max_norm=1.0)
    opt.step()
    twin = copy.deepcopy(opt)
    q = twin.param_groups[0]["params"][0]
    q.grad = p.grad.clone()
    opt.step()
    twin.step()
    assert torch.equal(p, q)
    where = opt.state[p]["exp_avg"].data_ptr(), opt.state[p]["step"].data_ptr()
    opt.load_state_dict(copy.deepcopy(twin.state_dict()))
    assert where == (opt.state[p]["exp_avg"].data_ptr(), opt.state[p]["step"].data_ptr())
    assert int(opt.state[p]["step"]) == 2


def test_parameters_that_were_moved(device):
    """A parameter taken to the host, or replaced by a view with gaps, after its first step: refused
    before any launch."""
    from gnnea import GnneaError
    from gnnea.optim import AdamW
    ps = [torch.nn.Parameter(torch.ones(6, 4, device=device)) for _ in range(2)]
    opt = AdamW(ps)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    ps[1].data = torch.ones(6, 8, device=device)[:, :4]
    ps[1].grad = torch.ones(6, 4, device=device)
    with pytest.raises(ValueError):
        opt.step()
    ps[1].grad = None
    ps[1].data = torch.ones(6, 4)
    ps[1].grad = torch.ones(6, 4)
    with pytest.raises(ValueError):
        opt.step()
    ps[0].grad = None
    with pytest.raises((GnneaError, ValueError)):
        opt.step()


def test_a_rate_that_was_replaced(device):
    """A rate set after the group was made is checked at the step, before any launch."""
    from gnnea.optim import AdamW
    p, q = (torch.nn.Parameter(torch.ones(5, device=device)) for _ in range(2))
    opt = AdamW([dict(params=[p]), dict(params=[q])], lr=torch.full((1,), 0.1, device=device))
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt.step()
    was = p.detach().clone(), int(opt.state[p]["step"])
    for lr in (torch.ones(1, device=device, dtype=torch.float64), torch.ones(1), -0.5,
               torch.ones(2, device=device)):
        opt.param_groups[1]["lr"] = lr
        with pytest.raises(ValueError):
            opt.step()
        assert torch.equal(p, was[0]) and int(opt.state[p]["step"]) == was[1]
