"""FlatAdamW at the edges of its formula: no eps, denominators next to nothing, 8-bit moments of bfloat16 parameters.

Tolerances: test_gpu_adamw.py, whose statement of the 8-bit format is used here."""
import pytest
import torch

from test_gpu_adamw import SIZES, U, _grads, _params

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
