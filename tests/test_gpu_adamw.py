"""FlatAdamW on the GPU (csrc/az_adamw.hip): against AdamW in 64 bits, the 8-bit moments bit for bit against their
definition, and the step inside a training loop.

Tolerances, u = 2^-24: m takes 3 roundings a step of terms that add to |b1 m| + |c1 g|; v takes 4; p takes the
roundings of p * keep (2) and of the update (at most 16: m's 3, v's 4 halved by the square root, sqrt, its product, eps,
step, the product, the division, the three scalars' own) of size |p| and |update|.  Over k steps they add up."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
GOLDEN, MASK = 0x9E3779B97F4A7C15, (1 << 64) - 1
SIZES = [(3, 5), (256,), (257,), (1,), (), (16, 2, 3, 3), (1000, 3), (255, 1), (40000,)]


def _params(sizes, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((0.1 * torch.randn(s, generator=g)).cuda().to(dtype)) for s in sizes]


def _grads(params, seed):
    g = torch.Generator().manual_seed(seed)
    return [(torch.exp(2 * torch.randn((), generator=g) - 4) * torch.randn(p.shape, generator=g) *
             (torch.rand(p.shape, generator=g) > 0.1)).cuda().to(p.dtype) for p in params]


class Exact:
    """AdamW in 64 bits, with the tolerances of its values."""

    def __init__(self, params):
        self.p = [p.detach().double().clone() for p in params]
        self.m, self.v = ([torch.zeros_like(p) for p in self.p] for _ in range(2))
        self.tp, self.tm, self.tv = ([torch.zeros_like(p) for p in self.p] for _ in range(3))
        self.t = 0

    def step(self, grads, lr, betas, eps, decay):
        self.t += 1
        b1, b2 = betas
        for i, g in enumerate(grads):
            g = g.double()
            self.tm[i] = b1 * self.tm[i] + 3 * U * (b1 * self.m[i].abs() + (1 - b1) * g.abs())
            self.tv[i] = b2 * self.tv[i] + 4 * U * (b2 * self.v[i] + (1 - b2) * g * g)
            self.m[i] = b1 * self.m[i] + (1 - b1) * g
            self.v[i] = b2 * self.v[i] + (1 - b2) * g * g
            step, root = lr[i] / (1 - b1 ** self.t), 1 / (1 - b2 ** self.t) ** 0.5
            den = self.v[i].sqrt() * root + eps
            up = step * self.m[i] / den
            # (the square root's slope: tv / (2 sqrt(v)), at most sqrt(tv) where v is next to nothing)
            rel = torch.minimum(self.tv[i] / (2 * self.v[i].sqrt() + 1e-300), self.tv[i].sqrt()) * root / den
            self.tp[i] = self.tp[i] + 2 * U * self.p[i].abs() + up.abs() * (16 * U + 2 * rel) + 2 * step * self.tm[i] / den + U * up.abs()
            self.p[i] = self.p[i] * (1 - lr[i] * decay[i]) - up

    def check(self, params, opt, half=0.0):
        m, v = opt.state_values()
        for i, (p, at) in enumerate(opt._places):
            k = next(j for j, q in enumerate(params) if q is p)
            off = (p.detach().double() - self.p[k]).abs() - (1 + half) * self.tp[k] - (half + U) * self.p[k].abs()
            assert bool((off <= 0).all()), ('p', k, off.max().item())
            if opt.state_bits == 32:
                for name, flat, want, tol in (('m', m, self.m, self.tm), ('v', v, self.v, self.tv)):
                    got = opt._cut(flat, p, at).double()
                    assert bool(((got - want[k]).abs() <= tol[k] + 1e-44).all()), (name, k)


@pytest.mark.parametrize('betas,eps', [((0.9, 0.999), 1e-8), ((0.0, 0.95), 1e-3), ((0.5, 0.0), 1e-8)])
def test_steps_match_adamw_in_64_bits(betas, eps):
    from alphazero_amd.optim import FlatAdamW
    params = _params(SIZES, 1)
    big = [i for i, p in enumerate(params) if p.dim() > 1]
    small = [i for i, p in enumerate(params) if p.dim() <= 1]
    ref = Exact(params)
    opt = FlatAdamW([dict(params=[params[i] for i in big], weight_decay=0.1), dict(params=[params[i] for i in small], lr=3e-2, weight_decay=0.0)],
                    lr=1e-2, betas=betas, eps=eps)
    sched = torch.optim.lr_scheduler.MultiStepLR(opt, [3], gamma=0.1)
    for k in range(6):
        grads = _grads(params, 10 + k)
        if k == 4:
            grads = [torch.zeros_like(g) for g in grads]
        for p, g in zip(params, grads):
            p.grad.copy_(g)
        rates = [g['lr'] for g in opt.param_groups]
        ref.step(grads, [rates[0] if i in big else rates[1] for i in range(len(params))], betas, eps, [0.1 if i in big else 0.0 for i in range(len(params))])
        opt.step()
        sched.step()
        ref.check(params, opt)
    assert opt.steps == 6
    inside = torch.zeros_like(opt.flat_p, dtype=torch.bool)
    for p, at in opt._places:
        inside[at:at + p.numel()] = True
    m, v = opt.state_values()
    assert not opt.flat_p[~inside].any() and not m[~inside].any() and not v[~inside].any()       # the gaps stay zero


def test_bfloat16_parameters_move_through_their_masters():
    """Steps far below bfloat16's resolution add up in the master; mixed types in one group; a weight written between
    two steps replaces its master."""
    from alphazero_amd.optim import FlatAdamW
    params = _params(SIZES, 2, torch.bfloat16) + _params([(7, 9), (300,)], 3)
    ref = Exact(params)
    opt = FlatAdamW(params, lr=1e-5, weight_decay=0.01)
    n = len(params)
    for k in range(20):
        grads = _grads(params, 40 + k)
        for p, g in zip(params, grads):
            p.grad.copy_(g)
        ref.step(grads, [1e-5] * n, (0.9, 0.999), 1e-8, [0.01] * n)
        opt.step()
    for p, at in opt._places:
        k = next(j for j, q in enumerate(params) if q is p)
        master = opt._cut(opt.flat_p, p, at)
        assert bool(((master.double() - ref.p[k]).abs() <= ref.tp[k] + U * ref.p[k].abs()).all())
        assert torch.equal(master.to(p.dtype), p.detach())
    with torch.no_grad():
        params[0].fill_(0.75)
    for p in params:
        p.grad.zero_()
    ref.p[0].fill_(0.75)
    ref.tp[0].zero_()
    ref.step([torch.zeros_like(p) for p in params], [1e-5] * n, (0.9, 0.999), 1e-8, [0.01] * n)
    opt.step()
    at = opt._places[[q is params[0] for q, _ in opt._places].index(True)][1]
    assert bool(((opt._cut(opt.flat_p, params[0], at).double() - ref.p[0]).abs() <= ref.tp[0] + U).all())


# ---- 8 bits: the definition, in numpy ----------------------------------------------------------------------------------
def _mix(z):
    z = ((z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9))
    z = ((z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB))
    return z ^ (z >> np.uint64(31))


def _random16(seed, t, blocks):
    with np.errstate(over='ignore'):
        key = _mix(np.array([(seed + GOLDEN * t) & MASK], np.uint64))
        z = _mix(np.arange(blocks * 128, dtype=np.uint64) * np.uint64(GOLDEN) + key).reshape(-1, 2, 1)
    r = (z >> np.array([0, 16, 32, 48], np.uint64)) & np.uint64(0xFFFF)
    return [r[:, k].reshape(blocks, 256).astype(np.int64) for k in (0, 1)]


def _encode(x, r, codes):
    """codes = 127 (m: the sign in bit 7) or 255 (v)."""
    a = np.abs(x).astype(np.float32).view(np.uint32).astype(np.int64)
    top = np.where(a.max(1) > 0x7F800000, 0x7FF, (a.max(1) + 0xFFFFF) >> 20)[:, None]
    q = np.where(a > 0x7F800000, 0x7FF, (a + (r << 4)) >> 20)
    lowest = np.maximum(top - (codes - 1), 1)
    if codes == 255:
        return np.where(a > 0, np.maximum(q, lowest) - (top - 255), 0).astype(np.uint8), top
    with np.errstate(invalid='ignore', over='ignore'):
        up = np.abs(x).astype(np.float64) * 131072 > (2 * r + 1) * (lowest << 20).astype(np.uint32).view(np.float32).astype(np.float64)
    k = np.where(q >= lowest, q - (top - 127), np.where(up, lowest - (top - 127), 0))
    return (k | np.where((x.view(np.uint32) >> 31 != 0) & (k > 0), 128, 0)).astype(np.uint8), top


def _decode(c, top, codes):
    k = (c & codes).astype(np.int64)
    x = (np.where(k > 0, k + top - codes, 0) << 20).astype(np.uint32).view(np.float32)
    return np.where(c > 127, -x, x) if codes == 127 else x


def _flat(opt):
    return opt.flat_g.cpu().numpy().reshape(-1, 256)


@pytest.mark.parametrize('sizes', [SIZES, [(1,)], [(700, 300)]])
def test_8_bit_moments_bit_for_bit(sizes):
    """Codes and tops after each of five steps against the definition; the parameters against 64 bits with the decoded
    moments as they were."""
    from alphazero_amd.optim import FlatAdamW
    params = _params(sizes, 4)
    opt = FlatAdamW(params, lr=1e-2, state_bits=8, seed=2 ** 63 + 12345)
    f = np.float32
    for k in range(5):
        for p, g in zip(params, _grads(params, 60 + k)):
            p.grad.copy_(g)
        g = _flat(opt)
        m0, v0 = (t.cpu().numpy().reshape(-1, 256) for t in opt.state_values())
        p0 = opt.flat_p.cpu().numpy().reshape(-1, 256)
        opt.step()
        m = m0 * f(0.9) + g * f(1 - 0.9)
        v = v0 * f(0.999) + (g * g) * f(1 - 0.999)
        rm, rv = _random16(opt.seed, k + 1, m.shape[0])
        cm, tm = _encode(m, rm, 127)
        cv, tv = _encode(v, rv, 255)
        assert np.array_equal(opt.codes_m.cpu().numpy().reshape(-1, 256), cm), k
        assert np.array_equal(opt.codes_v.cpu().numpy().reshape(-1, 256), cv), k
        assert np.array_equal(opt.tops.cpu().numpy().reshape(-1, 2), np.concatenate([tm, tv], 1)), k
        gm, gv = (t.cpu().numpy().reshape(-1, 256) for t in opt.state_values())
        assert np.array_equal(gm, _decode(cm, tm, 127)) and np.array_equal(gv, _decode(cv, tv, 255))
        # half a step of the leading bits on either side and no more: 2^-3 relative where a code exists
        far = np.abs(gm - m) > np.maximum(np.abs(m) * 2.0 ** -3, np.abs(m).max(1, keepdims=True) * 2.0 ** -15)
        assert not far.any()
        up = 1e-2 / (1 - 0.9 ** (k + 1)) * m.astype(np.float64) / (np.sqrt(v.astype(np.float64)) / np.sqrt(1 - 0.999 ** (k + 1)) + 1e-8)
        want = p0.astype(np.float64) * (1 - 1e-2 * 1e-2) - up
        assert np.all(np.abs(opt.flat_p.cpu().numpy().reshape(-1, 256) - want) <= 3 * U * np.abs(p0) + 16 * U * np.abs(up))


def test_8_bit_rounding_keeps_the_expectation():
    """4096 seeds, one step from zero: the mean of the decoded m of an element against m.  Rounding up by a step s with
    probability f has standard deviation s sqrt(f (1 - f)) <= s / 2 a draw; 5.5 standard deviations over 256 elements
    (4e-8 each) and the 2^-16 of the random numbers' own resolution."""
    from alphazero_amd.optim import FlatAdamW
    g = torch.Generator().manual_seed(3)
    grad = (torch.exp(2.5 * torch.randn(256, generator=g)) * torch.sign(torch.randn(256, generator=g))).cuda()
    p = [torch.nn.Parameter(torch.zeros(256, device='cuda'))]
    opt = FlatAdamW(p, state_bits=8)
    total, runs = torch.zeros(256, dtype=torch.float64, device='cuda'), 4096
    for seed in range(runs):
        opt.codes_m.zero_(), opt.codes_v.zero_(), opt.tops.zero_(), opt._step_dev.zero_()
        opt.seed = seed
        p[0].grad.copy_(grad)
        opt.step()
        total += opt.state_values()[0].double()
    m = (grad.float() * np.float32(1 - 0.9)).double()
    step = torch.maximum(m.abs() * 2.0 ** -3, m.abs().max() * 2.0 ** -15)
    assert bool(((total / runs - m).abs() <= step * (5.5 / 2 / runs ** 0.5 + 2.0 ** -15)).all())


def test_8_bit_extremes():
    """NaN and infinite gradients cost their element (as in 32 bits) and their block's moments, not the neighbours';
    zeros stay zero; subnormal and largest magnitudes keep their order."""
    from alphazero_amd.optim import FlatAdamW
    p = [torch.nn.Parameter(torch.ones(1024, device='cuda'))]
    opt = FlatAdamW(p, state_bits=8, weight_decay=0.0)
    g = torch.full((1024,), 1e-3, device='cuda')
    g[10], g[300], g[600] = float('nan'), float('inf'), 0.0
    p[0].grad.copy_(g)
    opt.step()
    m, v = opt.state_values()
    assert m[10].isnan() and v[10].isnan() and m[300].isinf() and v[300].isinf() and m[600] == 0 and v[600] == 0
    assert p[0][10].isnan() and p[0][300].isnan() and p[0][600] == 1 and bool(p[0][torch.arange(1024, device='cuda') // 256 == 3].isfinite().all())
    assert bool(m[512:].isfinite().all()) and bool((m[512:600] > 0).all())
    p[0].grad.zero_()
    opt.step()
    assert bool(p[0][512:].isfinite().all()) and bool(p[0][:10].isfinite().all()) and bool(p[0][256:300].isfinite().all())
    q = [torch.nn.Parameter(torch.zeros(256, device='cuda'))]
    opt = FlatAdamW(q, state_bits=8, weight_decay=0.0)
    q[0].grad.copy_(torch.logspace(-18, 18, 256).cuda())
    opt.step()
    m, v = opt.state_values()
    assert bool(m.isfinite().all()) and bool(v.isfinite().all()) and bool((v > 0).all()) and bool((v.diff() >= 0).all())


def test_8_bit_follows_a_change_that_nearest_rounding_would_swallow():
    """v after its gradients' size drops by 10: b2 = 0.999 moves v by a thousandth of itself a step, a hundredth of the
    3 bits' step.  After 2000 steps the mean of 4096 elements' v must have followed (0.135 of the old level is left; every
    element's noise is below half its value, the mean's below a 64th of that)."""
    from alphazero_amd.optim import FlatAdamW
    p = [torch.nn.Parameter(torch.zeros(4096, device='cuda'))]
    opt = FlatAdamW(p, state_bits=8, lr=0.0)
    sign = torch.sign(torch.randn(4096, device='cuda', generator=torch.Generator(device='cuda').manual_seed(1)))
    v = 0.0
    for k in range(4000):
        level = 1.0 if k < 2000 else 0.1
        if k in (0, 2000):
            p[0].grad.copy_(sign * level)
        opt.step()
        v = 0.999 * v + 0.001 * level ** 2
    got = opt.state_values()[1].double()
    assert abs(got.mean().item() / v - 1) < 6 * 0.5 / 64, (got.mean().item(), v)


# ---- state, captured steps, misuse -------------------------------------------------------------------------------------
def _train(opt, params, seeds):
    for s in seeds:
        for p, g in zip(params, _grads(params, s)):
            p.grad.copy_(g)
        opt.step()


@pytest.mark.parametrize('bits', [8, 32])
def test_state_dict_continues_the_run(bits, tmp_path):
    from alphazero_amd.optim import FlatAdamW
    a, b = ([*_params(SIZES, 5), *_params([(70, 5)], 6, torch.bfloat16)] for _ in range(2))
    oa, ob = (FlatAdamW(q, lr=1e-2, state_bits=bits, seed=9) for q in (a, b))
    _train(oa, a, range(3))
    torch.save({'model': [p.detach() for p in a], 'opt': oa.state_dict()}, tmp_path / 'c.pt')
    ck = torch.load(tmp_path / 'c.pt', weights_only=True)
    with torch.no_grad():
        for p, q in zip(b, ck['model']):
            p.copy_(q)
    ob.load_state_dict(ck['opt'])
    assert ob.steps == 3 and torch.equal(oa.flat_p, ob.flat_p)
    _train(oa, a, range(3, 6))
    _train(ob, b, range(3, 6))
    for x, y in ((oa.flat_p, ob.flat_p), (oa.flat_p16, ob.flat_p16), *zip(oa.state_values(), ob.state_values())):
        assert torch.equal(x, y)


def test_state_is_interchangeable_with_torch_adamw():
    from alphazero_amd.optim import FlatAdamW
    a, b, c = (_params(SIZES, 7) for _ in range(3))
    oa = torch.optim.AdamW(a, lr=1e-2)
    for s in range(3):
        for p, g in zip(a, _grads(a, s)):
            p.grad = g
        oa.step()
    ob, oc = FlatAdamW(b, lr=5.0), torch.optim.AdamW(c, lr=5.0)
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    ob.load_state_dict(oa.state_dict())
    assert ob.param_groups[0]['lr'] == 1e-2
    with torch.no_grad():
        for p, q in zip(a, c):
            q.copy_(p)
    oc.load_state_dict(ob.state_dict())
    for s in range(3, 6):
        for q in (a, b, c):
            for p, g in zip(q, _grads(q, s)):
                p.grad.copy_(g) if p.grad is not None else setattr(p, 'grad', g)
        for o in (oa, ob, oc):
            o.step()
    for x, y, z in zip(a, b, c):
        # (two float32 evaluations, 16 roundings of each of six updates of at most 3 lr)
        assert torch.allclose(x, y, rtol=1e-6, atol=200 * U * 1e-2) and torch.allclose(x, z, rtol=1e-6, atol=200 * U * 1e-2)
    o8 = FlatAdamW(_params(SIZES, 7), state_bits=8)
    o8.load_state_dict(ob.state_dict())
    for x, y in zip(o8.state_values(), ob.state_values()):
        x, y = x.reshape(-1, 256), y.reshape(-1, 256)
        low = y.abs().amax(1, keepdim=True) * 2.0 ** -15
        assert bool(((x - y).abs() <= torch.maximum(y.abs() * 2.0 ** -4 * 1.001, low)).all())   # to the nearest: half a step


def test_bad_state_is_refused():
    from alphazero_amd.optim import FlatAdamW
    p = _params([(4,), (5,)], 8)
    opt = FlatAdamW(p)
    _train(opt, p, range(1))
    sd = opt.state_dict()
    before = opt.state_values()[0].clone()
    for spoil in (lambda s: s['state'].pop(0), lambda s: s['state'][0].update(step=7), lambda s: s['state'][0].update(exp_avg=torch.zeros(3)),
                  lambda s: s['param_groups'][0].update(betas=(1.0, 0.9)), lambda s: s['param_groups'][0].update(amsgrad=True)):
        bad = opt.state_dict()
        spoil(bad)
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        assert torch.equal(opt.state_values()[0], before) and opt.steps == 1 and opt.param_groups[0]['betas'] == (0.9, 0.999)
    opt.load_state_dict(sd)
    assert torch.equal(opt.state_values()[0], before) and opt.steps == 1


@pytest.mark.parametrize('bits', [8, 32])
def test_captured_step_counts_on_and_follows_the_rate(bits):
    """One recorded step, replayed while the rate changes and with eager steps of the same optimizer in between, against
    an optimizer that takes every step eagerly: the same bits.  Two recorded optimizers take turns."""
    from alphazero_amd.optim import FlatAdamW
    pairs = []
    for seed in (1, 2):
        a, b = (_params(SIZES, seed) for _ in range(2))
        oa, ob = (FlatAdamW(q, lr=1e-2, state_bits=bits, seed=seed) for q in (a, b))
        oa.set_recorded_lr()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            oa.step_recorded()
        assert oa.steps == 0                                       # recording applies nothing
        pairs.append((a, oa, b, ob, graph))
    for k in range(8):
        for a, oa, b, ob, graph in pairs:
            lr = 1e-2 if k < 4 else 1e-3
            for q in (a, b):
                for p, g in zip(q, _grads(q, 100 + k)):
                    p.grad.copy_(g)
            for o in (oa, ob):
                o.param_groups[0]['lr'] = lr
            if k == 2:
                oa.step()
            else:
                oa.set_recorded_lr()
                graph.replay()
            ob.step()
            assert torch.equal(oa.flat_p, ob.flat_p) and all(torch.equal(x, y) for x, y in zip(oa.state_values(), ob.state_values())), k
    assert pairs[0][1].steps == 8


@pytest.mark.parametrize('bits', [8, 32])
def test_guard_withholds_the_whole_step(bits):
    from alphazero_amd.optim import FlatAdamW
    p = _params(SIZES, 9)
    opt = FlatAdamW(p, state_bits=bits)
    _train(opt, p, range(2))
    opt.set_recorded_lr()
    guard = torch.zeros(1, device='cuda')
    before = [t.clone() for t in (opt.flat_p, *opt.state_values())]
    for k, bad in enumerate((1e-6, 1.0, float('nan'), float('inf'))):
        guard.fill_(bad)
        opt.step_recorded(guard=guard)
        assert opt.steps == 2 and int(opt.withheld) == k + 1
        assert all(torch.equal(x, y) for x, y in zip(before, (opt.flat_p, *opt.state_values())))
    guard.fill_(5e-7)
    opt.step_recorded(guard=guard)
    assert opt.steps == 3 and int(opt.withheld) == 4 and not torch.equal(before[0], opt.flat_p)


def test_gradients_that_were_replaced_and_parameters_that_moved():
    from alphazero_amd._lib import AzError
    from alphazero_amd.optim import FlatAdamW
    a, b = (_params([(40, 3), (9,)], 11) for _ in range(2))
    oa, ob = FlatAdamW(a), FlatAdamW(b)
    grads = _grads(a, 1)
    for p, q, g in zip(a, b, grads):
        p.grad = g.clone()                                         # as after module.zero_grad() and a backward pass
        q.grad.copy_(g)
    oa.step(), ob.step()
    assert torch.equal(oa.flat_p, ob.flat_p) and all(p.grad is g for p, g in zip(a, oa._grads))
    oa.zero_grad()
    assert all(p.grad is g and not g.any() for p, g in zip(a, oa._grads))
    a[0].grad = None
    with pytest.raises(AzError, match='zero_grad'):
        oa.step()
    oa.zero_grad()
    b[1].data = b[1].data.clone()
    with pytest.raises(AzError, match='moved'):
        ob.step()
    with pytest.raises(ValueError, match='fixed'):
        oa.add_param_group(dict(params=_params([(3,)], 1)))
    for bad in ([torch.nn.Parameter(torch.zeros(3, device='cuda', dtype=torch.float16))],
                [torch.nn.Parameter(torch.zeros(3, device='cuda')), torch.nn.Parameter(torch.zeros(3))],
                [torch.nn.Parameter(torch.zeros(0, device='cuda'))]):
        with pytest.raises(ValueError):
            FlatAdamW(bad)
    with pytest.raises(ValueError, match='at most'):
        FlatAdamW([dict(params=[p]) for p in _params([(1,)] * 33, 1)])


def test_a_frozen_parameter_stays_and_a_closure_is_called():
    from alphazero_amd.optim import FlatAdamW
    p = _params([(5, 5), (6,)], 12)
    p[1].requires_grad_(False)
    frozen = p[1].detach().clone()
    opt = FlatAdamW(p, lr=0.1)

    def closure():
        opt.zero_grad()
        loss = p[0].square().sum()
        loss.backward()
        return loss
    first = opt.step(closure)
    assert float(opt.step(closure)) < float(first) and torch.equal(p[1], frozen) and 1 not in opt.state_dict()['state']


def test_settings_that_change_in_place():
    """A rate held in a tensor, as torch's schedulers fill it, and betas held in a list."""
    from alphazero_amd.optim import FlatAdamW
    a, b = (_params(SIZES, 21) for _ in range(2))
    rate, betas = torch.tensor(1e-2), [0.9, 0.999]
    oa, ob = FlatAdamW(a, lr=rate, betas=betas), FlatAdamW(b, lr=float(rate))
    for k in range(4):
        for q in (a, b):
            for p, g in zip(q, _grads(q, 30 + k)):
                p.grad.copy_(g)
        oa.step()
        ob.step()
        assert torch.equal(oa.flat_p, ob.flat_p), k
        rate.mul_(0.5)
        ob.param_groups[0]['lr'] = float(rate)
        if k == 1:
            betas[0] = 0.8
            ob.param_groups[0]['betas'] = (0.8, 0.999)


def test_channels_last_weights_keep_their_layout():
    from alphazero_amd.optim import FlatAdamW
    conv = torch.nn.Conv2d(8, 16, 3).cuda().to(memory_format=torch.channels_last)
    w = conv.weight.detach().clone(memory_format=torch.preserve_format)
    opt = FlatAdamW(conv.parameters())
    assert conv.weight.is_contiguous(memory_format=torch.channels_last) and torch.equal(conv.weight, w)
    assert conv.weight.grad.stride() == conv.weight.stride()
    conv(torch.randn(2, 8, 6, 7, device='cuda')).square().sum().backward()
    ref = torch.nn.Parameter(w.clone())
    ref.grad = conv.weight.grad.clone()
    opt.step()
    torch.optim.AdamW([ref]).step()
    assert torch.allclose(conv.weight, ref, rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize('bits', [8, 32])
def test_more_elements_than_32_bits_count(bits):
    """2^31 + 300 elements: the first and last ones against the formula, a second tensor behind them."""
    from alphazero_amd.optim import FlatAdamW
    n = 2 ** 31 + 300
    p = [torch.nn.Parameter(torch.zeros(n, device='cuda')), torch.nn.Parameter(torch.full((3,), 2.0, device='cuda'))]
    with torch.no_grad():
        p[0][-300:] = 1.0
    opt = FlatAdamW(p, lr=1e-2, weight_decay=0.1, state_bits=bits)
    assert opt._places[1][1] > 2 ** 31
    p[0].grad[-300:] = torch.linspace(-1, 1, 300, device='cuda')
    p[1].grad.fill_(-3.0)
    opt.step()
    g = torch.linspace(-1, 1, 300, device='cuda').double()
    want = 1 - 1e-3 - 1e-2 * g / (g.abs() + 1e-8)
    assert bool(((p[0][-300:].double() - want).abs() <= 20 * U).all()) and not p[0][:1000].any()
    assert bool(((p[1].double() - (2 * (1 - 1e-3) + 1e-2)).abs() <= 24 * U).all())
    m, _ = opt.state_values()
    at = opt._places[1][1]
    assert bool(((m[at:at + 3] + 0.3).abs() <= (0.3 * 2 ** -3 if bits == 8 else 1e-7)).all())
    del m
    opt.step()
    assert opt.steps == 2


def test_another_stream():
    from alphazero_amd.optim import FlatAdamW
    a, b = (_params(SIZES, 13) for _ in range(2))
    oa, ob = FlatAdamW(a, state_bits=8), FlatAdamW(b, state_bits=8)
    side = torch.cuda.Stream()
    for k in range(3):
        for p, q, g in zip(a, b, _grads(a, k)):
            p.grad.copy_(g), q.grad.copy_(g)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            oa.step()
        torch.cuda.current_stream().wait_stream(side)
        ob.step()
    assert torch.equal(oa.flat_p, ob.flat_p) and torch.equal(oa.codes_v, ob.codes_v)


# ---- the operators together, as a training job uses them ----------------------------------------------------------------
def _job(norm, bits, **kw):
    from alphazero_amd.config import AlphaZeroConfig
    return AlphaZeroConfig(conf={
        'game': {'module': 'alphazero.games.connectfour', 'name': 'ConnectFour'},
        'model': {'module': 'alphazero.games.connectfour', 'name': 'AlphaZeroC4',
                  'kwargs': {'num_blocks': 2, 'channels_per_block': 32, 'norm': norm}},
        'loss': {'module': 'alphazero.loss', 'name': 'AlphaZeroLoss'},
        'training': dict({'num_steps': 12, 'batch_size': 32, 'lr': 1e-3, 'momentum': 0.9, 'weight_decay': 1e-2, 'lr_schedule_gamma': 0.1,
                          'lr_schedule': [6], 'optimizer': 'adamw', 'state_bits': bits}, **kw),
        'selfplay': {'num_expansions_per_sim': 8, 'exploration_depth': 4, 'reuse_search_tree': True}})


def _window(dev):
    from alphazero_amd import engine as E
    from alphazero_amd.games import ConnectFour
    from alphazero_amd.replay_buffer import DeviceReplayWindow
    eng = E.SelfPlayEngine(E._lib.GAME_C4, 256, 16, exploration_depth=4, reuse_search_tree=True, seed=5, device=0)
    window = DeviceReplayWindow(ConnectFour, 4096, dev)
    while len(window) < 512:
        eng.begin_move_uniform(); eng.run_sims_uniform(16); eng.choose_and_advance()
        window.add_records(eng.drain_finished_bytes())
    return window


class _Server:
    def update(self, model, version):
        pass


class _Writer:
    def __init__(self):
        self.rows = []

    def add_scalar(self, tag, value, step):
        self.rows.append((tag, float(value), int(step)))


@pytest.mark.parametrize('norm,bits,record', [('group', 32, True), ('group', 8, True), ('group', 8, False), ('batch', 8, True)])
def test_training_worker_with_group_norm_and_adamw(norm, bits, record):
    """Ten steps of TrainingWorker, three eager and the rest replayed (or all eager), each checked from its own start: the
    logged losses against the network with the weights before the step on the same batch, the gradients against autograd
    there, and the update against an optimizer of the same state that steps eagerly on the same gradients: the same bits.
    (Two trainings are not compared: the library's convolutions add in no fixed order, and Adam turns the last bits of
    a gradient next to zero into a step of the full rate.)  A loss is a mean of values below 5 whose logits went through
    7 layers of sums of up to 288 terms, each off by at most 288 u of its magnitudes: 7 * 288 * u * 5 < 1e-3; a gradient
    passes twice as many and is a sum over 32 boards of 42 cells: 1e-2 of its norm."""
    import copy
    from alphazero_amd.loss import masked_cross_entropy
    from alphazero_amd.optim import FlatAdamW
    from alphazero_amd.training import TrainingWorker
    dev = torch.device('cuda:0')
    window = _window(dev)
    torch.manual_seed(11)
    writer = _Writer()
    tw = TrainingWorker(_job(norm, bits), _Server(), window, writer, dev, record_step=record)
    opt = tw._optimizer
    assert isinstance(opt, FlatAdamW) and (tw._hand is not None) == (norm == 'batch')
    taken, batch = [], tw._batch
    tw._batch = lambda: taken.append(batch()) or taken[-1]
    for k in range(10):
        before = copy.deepcopy(tw.model.state_dict())
        state = opt.state_dict()
        writer.rows.clear()
        assert tw.process_batch() == k + 1
        recorded = record and k >= tw.EAGER_STEPS
        x, p, z, valid = (tw._gx, tw._gp, tw._gz, tw._gvalid) if recorded else taken[-1][:4]
        shadow = tw._config.Model().to(dev)
        shadow.load_state_dict(before)
        shadow.train()
        other = FlatAdamW(shadow.parameters(), state_bits=bits)
        logits, v = shadow(x, valid.bool())
        policy, value = masked_cross_entropy(logits, p, valid.bool()).mean(), ((z.reshape(-1, 1) - v) ** 2).mean()
        (policy + value).backward()
        logged = {r[0]: r[1] for r in writer.rows}
        assert abs(logged['loss/policy'] - policy.item()) < 1e-3 and abs(logged['loss/value'] - value.item()) < 1e-3, k
        for (name, a), b in zip(tw.model.named_parameters(), shadow.parameters()):
            if norm == 'batch' and name == '_policy_head._cbr.0.bias':
                continue                                           # (zero but for rounding: batch-norm takes the bias out)
            assert (a.grad - b.grad).norm() <= 1e-2 * b.grad.norm() + 1e-6, (k, name)
        other.load_state_dict(state)
        other.flat_g.copy_(opt.flat_g)
        other.step()
        assert torch.equal(other.flat_p, opt.flat_p) and all(torch.equal(a, b) for a, b in zip(other.state_values(), opt.state_values())), k
    assert (tw._graph is not None) == record and opt.steps == 10 and abs(opt.param_groups[0]['lr'] - 1e-4) < 1e-12


def test_a_writer_may_keep_what_it_is_given():
    """The losses of the eager steps, kept as tensors, hold no graph of the parameters when the step is recorded."""
    from alphazero_amd.training import TrainingWorker

    class Keeper:
        kept = []

        def add_scalar(self, tag, value, step):
            self.kept.append(value)
    dev = torch.device('cuda:0')
    tw = TrainingWorker(_job('group', 32), _Server(), _window(dev), Keeper(), dev)
    for _ in range(tw.EAGER_STEPS):
        tw.process_batch()
    tensors = [v for v in Keeper.kept if torch.is_tensor(v)]
    assert tensors and all(v.grad_fn is None for v in tensors)
    for _ in range(3):
        tw.process_batch()
    assert tw._graph is not None and tw._optimizer.steps == 6


def test_recorded_step_of_a_bad_batch_is_withheld():
    from alphazero_amd.training import TrainingWorker
    dev = torch.device('cuda:0')
    window = _window(dev)
    torch.manual_seed(3)
    tw = TrainingWorker(_job('group', 8), _Server(), window, None, dev)
    for _ in range(5):
        tw.process_batch()
    before = tw._optimizer.flat_p.clone()
    window.p.mul_(1.5)
    with pytest.raises(AssertionError, match='valid distribution'):
        for _ in range(2 * tw.CHECK_EVERY):
            tw.process_batch()
    assert torch.equal(tw._optimizer.flat_p, before) and tw._optimizer.steps == 5


def test_group_normalised_network_plays_and_trains():
    """synchronous_play_and_train with norm='group' and 8-bit AdamW: self-play evaluates the torch module with the
    group norm kernels, the trainer steps, versions reach the worker."""
    from alphazero_amd.train import synchronous_play_and_train
    server, worker, trainer = synchronous_play_and_train(_job('group', 8, num_steps=6), torch.device('cuda:0'), num_games=256, num_steps=6, seed=1)
    assert server._version == 6 and trainer._optimizer.steps == 6 and worker._fused is None
    for k, v in trainer.model.state_dict().items():
        assert bool(v.isfinite().all()), k
    worker.refresh_model()
    worker.play_move(False)
    assert worker.engine.stats()['errors'] == 0


def test_search_of_one_game_with_a_group_normalised_network():
    """run_mcts evaluates one position at a time: the same visits as with the network's torch statement on the CPU would
    need equal float32 sums, so what is checked is the evaluation, 1e-5 of the CPU statement, and that the search runs."""
    from alphazero_amd.games import ConnectFour
    from alphazero_amd.mcts import MCTreeNode, evaluate, run_mcts
    from alphazero_amd.models import AlphaZeroC4
    torch.manual_seed(2)
    cpu = AlphaZeroC4(3, 32, norm='group').eval()
    gpu = AlphaZeroC4(3, 32, norm='group').eval()
    gpu.load_state_dict(cpu.state_dict())
    gpu.cuda()
    game = ConnectFour()
    for a in (3, 3, 2):
        p0, v0 = evaluate(game, cpu)
        p1, v1 = evaluate(game, gpu)
        assert np.allclose(p0, p1, atol=1e-5) and np.allclose(v0, v1, atol=1e-5)
        game.take_action(a)
    root = MCTreeNode()
    np.random.seed(0)
    run_mcts(game, root, gpu, 24)
    assert int(root.num_visits.sum()) == 24
