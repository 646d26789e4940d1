"""Group norm: calls that reach its autograd function in other ways than a plain forward and backward pass.

Tolerances and their derivation: test_gpu_norm.py, whose reference and check are used here; where a test compares two calls
of the kernels on the same values, the bits are equal."""
import pytest
import torch

from test_gpu_norm import _check, _inputs, _reference, _run

pytestmark = pytest.mark.gpu


def _grads(x, groups, w, b, r, dy, act='relu'):
    from alphazero_amd.norm import group_norm_act
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], act=act, residual=leaves[3])
    return torch.autograd.grad(y, leaves, dy)


def _pinned():
    return torch.autograd.graph.save_on_cpu(pin_memory=True)


def _plain_order():
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.contiguous())


def _every_second():
    """The values in every second place of a larger buffer."""
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0])


@pytest.mark.parametrize('hooks', [_pinned, _plain_order, _every_second])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(6, 32, 4, 6, 7), (2, 64, 8, 32, 32), (3, 320, 32, 64, 64)])
def test_saved_tensors_that_come_back_in_another_layout(hooks, dtype, shape):
    """A saved-tensor hook may return the same values in another order of memory."""
    n, c, groups, h, w = shape
    x, wt, b, r, dy = _inputs(n, c, h, w, dtype, torch.float32, True, 31)
    want = _grads(x, groups, wt, b, r, dy)
    with hooks():
        got = _grads(x, groups, wt, b, r, dy)
    assert all(torch.equal(g, e) for g, e in zip(got, want))
    assert got[0].is_contiguous(memory_format=torch.channels_last) and got[3].is_contiguous(memory_format=torch.channels_last)


@pytest.mark.parametrize('other', [lambda t: t[:1], lambda t: t.half(), lambda t: t.cpu(), lambda t: t.double().float().unsqueeze(0)])
def test_saved_tensors_that_come_back_as_others_are_refused(other):
    x, wt, b, r, dy = _inputs(6, 32, 6, 7, torch.float32, torch.float32, True, 32)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other), pytest.raises(RuntimeError, match='came back as another one'):
        _grads(x, 4, wt, b, r, dy)


def test_forward_mode_tangents_are_refused():
    """In x, and in the gradient that comes into the backward pass; a batch of such gradients likewise.  Calls without them
    go on as before."""
    import torch.autograd.forward_ad as forward_ad
    from alphazero_amd.norm import group_norm_act
    x, wt, b, r, dy = _inputs(3, 16, 6, 7, torch.float32, torch.float32, True, 33)
    want = _run(x, 4, wt, b, r, dy, 'relu')
    with forward_ad.dual_level():
        with torch.no_grad(), pytest.raises(NotImplementedError, match='forward-mode'):
            group_norm_act(forward_ad.make_dual(x, torch.ones_like(x)), 4, wt, b, residual=r)
        leaf = x.detach().requires_grad_()
        y = group_norm_act(leaf, 4, wt, b, residual=r)
        with pytest.raises(NotImplementedError, match='forward-mode'):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(dy, torch.ones_like(dy)))
        y = group_norm_act(leaf, 4, wt, b, residual=r)
        assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want['dx'])
    y = group_norm_act(leaf, 4, wt, b, residual=r)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.autograd.grad(y, leaf, torch.stack([dy, dy]), is_grads_batched=True)


@pytest.mark.filterwarnings('ignore')
def test_tracing_is_refused_and_leaves_nothing_behind():
    from torch.fx.experimental.proxy_tensor import make_fx
    from alphazero_amd.norm import GroupNormAct, group_norm_act
    x, wt, b, r, dy = _inputs(3, 16, 6, 7, torch.float32, torch.float32, True, 34)
    want = group_norm_act(x, 4)
    module = GroupNormAct(4, 16).cuda()
    for trace in (lambda: torch.jit.trace(lambda t: group_norm_act(t, 4), (x,), check_trace=False), lambda: torch.jit.trace(module, (x,)),
                  lambda: make_fx(lambda t: group_norm_act(t, 4))(x), lambda: make_fx(lambda t: module(t))(x)):
        with pytest.raises(NotImplementedError, match='traced'):
            trace()
        assert torch.equal(group_norm_act(x, 4), want)
    leaf = x.detach().requires_grad_()
    y = group_norm_act(leaf, 4, wt, b, residual=r)
    with pytest.raises(NotImplementedError, match='traced'):
        make_fx(lambda t: torch.autograd.grad(y, leaf, t, retain_graph=True)[0])(dy)
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], _run(x, 4, wt, b, r, dy, 'relu')['dx'])


@pytest.mark.parametrize('h,w', [(46340, 46340), (1, 2 ** 31 - 1)])
def test_the_longest_samples(h, w):
    """One channel of up to 2^31 - 1 values, all zero but for the last thousand, gradients there and in the first thousand.
    Sums of the definition are those of the values that are not zero."""
    from alphazero_amd.norm import group_norm_act
    n, k = h * w, 1000
    g = torch.Generator(device='cuda').manual_seed(35)
    head, tail = (torch.randn(k, device='cuda', generator=g).bfloat16() for _ in range(2))
    values = torch.randn(k, device='cuda', generator=g).bfloat16()
    x, dy = (torch.zeros(1, 1, h, w, dtype=torch.bfloat16, device='cuda') for _ in range(2))
    x.view(-1)[-k:] = values
    dy.view(-1)[:k], dy.view(-1)[-k:] = head, tail
    wt, b = torch.full((1,), 1.5, device='cuda', requires_grad=True), torch.full((1,), 0.25, device='cuda', requires_grad=True)
    x.requires_grad_()
    y = group_norm_act(x, 1, wt, b, act='none')
    dx, dw, db = torch.autograd.grad(y, [x, wt, b], dy)
    v, dh, dt = values.double(), head.double(), tail.double()
    mean = v.sum() / n
    rstd = 1 / torch.sqrt((v * v).sum() / n - mean * mean + 1e-5)
    at_zero, at_v = -mean * rstd, (v - mean) * rstd
    half = 2.0 ** -8
    yv = y.detach().view(-1)
    assert bool(((yv[-k:].double() - (1.5 * at_v + 0.25)).abs() <= half * (1.5 * at_v + 0.25).abs() + 1e-6 * (at_v.abs() + 1)).all())
    assert bool((yv[:-k] == yv[0]).all()) and abs(yv[0].double() - (1.5 * at_zero + 0.25)) <= half
    # (sums of 2000 terms, each rounded four times, in chains of no more than that)
    terms, tol = torch.cat([dh * at_zero, dt * at_v]), 2010 * 2.0 ** -24
    assert abs(dw[0].double() - terms.sum()) <= tol * terms.abs().sum()
    assert abs(db[0].double() - (dh.sum() + dt.sum())) <= tol * (dh.abs().sum() + dt.abs().sum())
    ma, mx = 1.5 * (dh.sum() + dt.sum()) / n, 1.5 * terms.sum() / n
    for got, d, xhat in ((dx.view(-1)[:k], dh, at_zero), (dx.view(-1)[-k:], dt, at_v)):
        want = rstd * (1.5 * d - ma - xhat * mx)
        assert bool(((got.double() - want).abs() <= half * want.abs() + 1e-5 * rstd * (d.abs() + 1e-3)).all())


def test_more_channels_than_one_launch_of_parameter_gradients_takes():
    """2^25 + 24 channels: two columns each for dweight and dbias.  Every group is the same eight values in another order of
    channels' gradients, so the definition is that of one group."""
    from alphazero_amd.norm import group_norm_act
    c, groups = 2 ** 25 + 24, (2 ** 25 + 24) // 8
    one = torch.tensor([-2.0, -1.0, -0.5, 0.0, 0.25, 0.5, 1.0, 3.0], device='cuda')
    x = one.repeat(groups)[None].repeat(2, 1)
    x[1] *= 2
    x.requires_grad_()
    wt, b = (torch.full((c,), v, device='cuda', requires_grad=True) for v in (1.0, 0.0))
    scale = 1 + (torch.arange(c, device='cuda') % 1000).float() / 1000
    dy = torch.stack([scale, -2 * scale])
    dw, db = torch.autograd.grad(group_norm_act(x, groups, wt, b, act='none'), [wt, b], dy)
    xhat = torch.stack([(k * one.double() - k * one.double().mean()) / torch.sqrt(k * k * one.double().var(correction=0) + 1e-5) for k in (1, 2)])
    want = (xhat[0] - 2 * xhat[1]).repeat(groups) * scale.double()
    assert bool(((dw.double() - want).abs() <= 20 * 2.0 ** -24 * 3 * xhat.abs().max() * scale).all())
    assert torch.equal(db, -scale)


@pytest.mark.parametrize('shape', [(1, 255, 1024, 1024), (40000, 3, 19, 19)])
def test_long_sums_of_equal_terms(shape):
    """Equal gradients, whose float32 sum is rounded the same way at every step: n of them added in one chain are off by n / 6
    half steps.  2048 rows at most are added so, the rest in 64 bits."""
    from alphazero_amd.norm import group_norm_act
    n, c, h, w = shape
    x = torch.zeros(shape, device='cuda').contiguous(memory_format=torch.channels_last)
    b = torch.zeros(c, device='cuda', requires_grad=True)
    dy = torch.full_like(x, 0.3)
    (db,) = torch.autograd.grad(group_norm_act(x, 1, None, b, act='none'), [b], dy)
    want = n * h * w * dy[0, 0, 0, 0].double()
    assert bool(((db.double() - want).abs() <= (2048 + 1) * 2.0 ** -24 * want).all())


@pytest.mark.parametrize('shape', [(3, 32, 4, 6, 7), (2, 30, 5, 5, 3), (3, 48, 4, 19, 19), (2, 64, 8, 32, 32), (1, 320, 32, 64, 64), (4, 24, 4, 1, 1)])
@pytest.mark.parametrize('offset', [1e5, -1e6])
@pytest.mark.parametrize('act', ['none', 'relu'])
def test_means_that_are_large_against_the_spread(shape, offset, act):
    """float32 values 10^5 and 10^6 spreads from zero, within the tolerances of any others."""
    n, c, groups, h, w = shape
    x, wt, b, r, dy = _inputs(n, c, h, w, torch.float32, torch.float32, True, 36, offset)
    want, tol = _reference(x, groups, wt, b, r, dy, act)
    _check(_run(x, groups, wt, b, r, dy, act), want, tol, torch.float32, torch.float32)


@pytest.mark.parametrize('shape', [(4, 16, 2, 6, 7), (2, 64, 8, 32, 32), (1, 6, 2, 100, 101), (5, 8, 1, 1, 1)])
@pytest.mark.parametrize('value', [1.0, -12345.678, 1e-3])
def test_groups_equal_but_for_one_last_bit_without_an_eps(shape, value):
    """eps = 0 and one value a half step away: the variance is (n - 1) / n^2 of that step's square and not zero."""
    n, c, groups, h, w = shape
    x = torch.full((n, c, h, w), value, device='cuda').contiguous(memory_format=torch.channels_last)
    per = c // groups
    for g in range(groups):
        for s in range(n):                                             # the first value of the group, the last, one within
            at = (g * per + (0, per - 1, per // 2)[s % 3], (0, h - 1, h // 2)[s % 3], (0, w - 1, w // 2)[s % 3])
            x[s][at] = torch.nextafter(x[s][at], torch.tensor(float('inf' if s % 2 else '-inf'), device='cuda'))
    wt, b, dy = torch.ones(c, device='cuda'), torch.zeros(c, device='cuda'), torch.randn(n, c, h, w, device='cuda').contiguous(memory_format=torch.channels_last)
    # The reference goes by x less `value`, which is exact and changes nothing: the mean of x itself lies a thousandth of a half
    # step from `value`, and no 64-bit number is nearer to it than 2^-53 of it.  That is what the kernel's mean is off by (half
    # a unit in the last place, where the first value and the mean's distance from it are added), and y by as much times
    # rstd: n / sqrt(n - 1) over the step of at least 2^-24 |value| makes it 2^-29 sqrt(n), some 2^-24 of values of 1 / sqrt(n).
    want, tol = _reference(x - x.new_tensor(value), groups, wt, b, None, dy, 'none', eps=0.0)
    got = _run(x, groups, wt, b, None, dy, 'none', eps=0.0)
    count = per * h * w
    tol['y'] = tol['y'] + 2.0 ** -29 * count / (count - 1) ** 0.5
    assert all(bool(v.isfinite().all()) for v in got.values())
    _check(got, want, tol, torch.float32, torch.float32)


def test_a_first_value_far_from_its_group():
    """Sums are taken from the group's first value: here it lies a million spreads of the others away."""
    x, wt, b, r, dy = _inputs(4, 32, 6, 7, torch.float32, torch.float32, True, 37)
    x[:, ::8, 0, 0] = torch.tensor([1e6, -1e6, 1e3, -3e4], device='cuda')[:, None]
    want, tol = _reference(x, 4, wt, b, r, dy, 'relu')
    _check(_run(x, 4, wt, b, r, dy, 'relu'), want, tol, torch.float32, torch.float32)


@pytest.mark.parametrize('dtype,param', [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize('shape', [(6, 32, 4, 6, 7), (2, 64, 8, 32, 32), (3, 48, 4, 19, 19), (3, 320, 32, 64, 64)])
@pytest.mark.parametrize('act', ['relu', 'silu'])
def test_weight_and_bias_off_any_border(dtype, param, shape, act):
    """Both, or one of them, one value off a 16-byte border, as in a buffer without gaps: the bits of aligned ones."""
    n, c, groups, h, w = shape
    x, wt, b, r, dy = _inputs(n, c, h, w, dtype, param, True, 38)
    want = _run(x, groups, wt, b, r, dy, act)
    odd = lambda t, k: torch.empty(c + 8, dtype=param, device='cuda')[k:k + c].copy_(t)
    for kw, kb in ((1, 1), (3, 0), (0, 1)):
        got = _run(x, groups, odd(wt, kw), odd(b, kb), r, dy, act)
        assert all(torch.equal(got[k], want[k]) for k in want), (kw, kb)


@pytest.mark.parametrize('gain', [2.0 ** 120, 2.0 ** 60, 2.0 ** -60, 2.0 ** -120])
@pytest.mark.parametrize('shape', [(3, 32, 4, 6, 7), (3, 48, 4, 19, 19), (1, 320, 32, 64, 64)])
def test_the_ends_of_the_range(shape, gain):
    n, c, groups, h, w = shape
    x, wt, b, r, dy = _inputs(n, c, h, w, torch.float32, torch.float32, True, 39, 0.0, gain)
    for act in ('relu', 'silu'):
        want, tol = _reference(x, groups, wt, b, r, dy, act, eps=0.0)
        _check(_run(x, groups, wt, b, r, dy, act, eps=0.0), want, tol, torch.float32, torch.float32)
