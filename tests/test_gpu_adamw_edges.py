"""FlatAdamW at the edges of its formula: no eps, denominators next to nothing, 8-bit moments of bfloat16 parameters.

Tolerances: test_gpu_adamw.py, whose statement of the 8-bit format is used here."""
import numpy as np
import pytest
import torch

from test_gpu_adamw import SIZES, U, _decode, _encode, _grads, _params, _random16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_without_an_eps_what_never_had_a_gradient_stays(bits, dtype):
    """eps = 0: 0 / 0 counts as no update, in the gaps between tensors, which have to stay zero, and in elements whose
    gradients were all zero (there torch.optim.AdamW's become NaN).  The others follow the formula."""
    from alphazero_amd.optim import FlatAdamW
    params = _params(SIZES, 3, dtype)
    start = [p.detach().clone() for p in params]
    grads = _grads(params, 4)
    opt = FlatAdamW(params, lr=1e-2, eps=0.0, weight_decay=0.1, state_bits=bits)
    for k in range(3):
        for p, g in zip(params, grads):
            p.grad.copy_(g)
        opt.step()
    inside = torch.zeros_like(opt.flat_p, dtype=torch.bool)
    for p, at in opt._places:
        inside[at:at + p.numel()] = True
    m, v = opt.state_values()
    assert not opt.flat_p[~inside].any() and not m[~inside].any() and not v[~inside].any()
    assert opt.flat_p16 is None or not opt.flat_p16[~inside].any()
    assert bool(opt.flat_p.isfinite().all())
    keep = (1 - 1e-2 * 0.1) ** 3
    for (p, at), p0, g in zip(opt._places, start, grads):
        idle = g == 0
        value = opt._cut(opt.flat_p, p, at).double()
        # (three products of three roundings each)
        assert bool(((value - p0.double() * keep)[idle].abs() <= 10 * U * p0.double().abs()[idle]).all())
        if bits == 32:
            # (the same gradient three times: m and v over their corrections are g and g^2, every update lr in size)
            want, size = p0.double(), (1e-2 * torch.sign(g.double()))
            for _ in range(3):
                want = want * (1 - 1e-2 * 0.1) - size
            assert bool(((value - want)[~idle].abs() <= 3 * 20 * U * (p0.double().abs() + 0.03)[~idle]).all())


@pytest.mark.parametrize('eps', [2.0 ** -40, 2.0 ** -36, 1e-10, 1e-8])
@pytest.mark.parametrize('betas', [(0.9, 0.999), (0.9, 0.9999999), (0.9, 0.5)])
def test_second_moments_below_the_smallest_normal_number(eps, betas):
    """v is subnormal after a first gradient of 10^-18, and its root, over the correction, is as large as the gradient:
    4e-6 of an eps of 2^-40.  p starts at 0, so that the update is the result: 16 roundings of it, and those of v (four; its
    last bit is 2^-149, and the smallest v that is looked at 2^-130)."""
    from alphazero_amd.optim import FlatAdamW
    p = [torch.nn.Parameter(torch.zeros(1024, device='cuda'))]
    opt = FlatAdamW(p, lr=1.0, betas=betas, eps=eps, weight_decay=0.0)
    c2 = 1 - betas[1]
    g = torch.logspace(np.log10(2.0 ** -65 / c2 ** 0.5), np.log10(2.0 ** -60 / c2 ** 0.5), 1024).cuda()
    p[0].grad.copy_(g)
    opt.step()
    want = -g.double() / (g.double() + eps)
    # (g's own square, rounded, against the last bit of a subnormal number: 2^-20 of v at 2^-130, half of that in its root)
    assert bool(((p[0].detach().double() - want).abs() <= (20 * U + 2.0 ** -21 * g.double() / (g.double() + eps)) * want.abs()).all())


@pytest.mark.parametrize('sizes', [SIZES, [(700, 300)]])
def test_8_bit_moments_of_bfloat16_parameters_bit_for_bit(sizes):
    """Codes and tops after each of five steps against the definition, from bfloat16 gradients; the masters against 64 bits, the
    parameters their roundings."""
    from alphazero_amd.optim import FlatAdamW
    params = _params(sizes, 4, torch.bfloat16)
    opt = FlatAdamW(params, lr=1e-2, state_bits=8, seed=2 ** 62 + 99)
    f = np.float32
    rows = lambda t: t.float().cpu().numpy().reshape(-1, 256)
    for k in range(5):
        for p, g in zip(params, _grads(params, 60 + k)):
            p.grad.copy_(g)
        g, p0 = rows(opt.flat_g16), rows(opt.flat_p)
        m0, v0 = (rows(t) for t in opt.state_values())
        opt.step()
        m = m0 * f(0.9) + g * f(1 - 0.9)
        v = v0 * f(0.999) + (g * g) * f(1 - 0.999)
        rm, rv = _random16(opt.seed, k + 1, m.shape[0])
        cm, tm = _encode(m, rm, 127)
        cv, tv = _encode(v, rv, 255)
        assert np.array_equal(opt.codes_m.cpu().numpy().reshape(-1, 256), cm), k
        assert np.array_equal(opt.codes_v.cpu().numpy().reshape(-1, 256), cv), k
        assert np.array_equal(opt.tops.cpu().numpy().reshape(-1, 2), np.concatenate([tm, tv], 1)), k
        gm, gv = (rows(t) for t in opt.state_values())
        assert np.array_equal(gm, _decode(cm, tm, 127)) and np.array_equal(gv, _decode(cv, tv, 255))
        up = 1e-2 / (1 - 0.9 ** (k + 1)) * m.astype(np.float64) / (np.sqrt(v.astype(np.float64)) / np.sqrt(1 - 0.999 ** (k + 1)) + 1e-8)
        want = p0.astype(np.float64) * (1 - 1e-2 * 1e-2) - up
        assert np.all(np.abs(rows(opt.flat_p) - want) <= 3 * U * np.abs(p0) + 16 * U * np.abs(up))
        assert torch.equal(opt.flat_p.to(torch.bfloat16), opt.flat_p16)
