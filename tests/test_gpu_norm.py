"""Group norm with activation and residual sum on the GPU (csrc/az_norm.hip) against the formulas in 64 bits.

Tolerances, counted in roundings (u = 2^-24; h = half a step of the output's type: 2^-24, 2^-8, 2^-11):
  y   x - mean (two subtractions), rstd, their product, the product with w, two sums: at most 8 u (|xhat w| + |b| + |res|);
      silu adds exp and a division, 8 u (|z| + 1) for a slope of at most 1.1; then h |y|
  dx  a = dz w has 4 roundings of its own (silu: 24, of factors that are at most 1.1 |dy|), the two means are sums of
      terms rounded 4 (28) times each, added in 32 bits in chains of at most L: dx is off by at most
      rstd u ((8 + s) |a| + (L + 8 + s) (mean|a| + |xhat| mean|a xhat|)), s = 0 (24); then h |dx|
  dw, db  (L + 8 + s) u sum|dz xhat|, (L + 8 + s) u sum|dz|; then h of the parameter's type
L: a thread adds at most the rows of its column that its workgroup holds, min(N * cells, 2048)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _inputs(n, c, h, w, dtype, param, residual, seed, offset=0.0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    cl = lambda t: t.cuda().to(dtype).contiguous(memory_format=torch.channels_last)
    x = cl(gain * rnd(n, c, h, w) * torch.exp(0.3 * rnd(c)).view(1, c, 1, 1) + offset)
    wt, b = (1 + 0.3 * rnd(c)).cuda().to(param), (0.3 * rnd(c)).cuda().to(param)
    r = cl(rnd(n, c, h, w).relu()) if residual else None
    dy = cl(rnd(n, c, h, w))
    return x, wt, b, r, dy


def _act(z, act):
    return torch.where(z > 0, z, torch.zeros_like(z)) if act == 'relu' else z * torch.sigmoid(z) if act == 'silu' else z


def _reference(x, groups, w, b, r, dy, act, eps=1e-5):
    """Everything in 64 bits by the formulas (the gradients are checked against differences below), with the sums of
    magnitudes that the tolerances are made of."""
    n, c, h, ww = x.shape
    d = lambda t: t.detach().double()
    rows = d(x).reshape(n, groups, -1)
    mean = rows.mean(2, keepdim=True)
    rstd = 1 / torch.sqrt(((rows - mean) ** 2).mean(2, keepdim=True) + eps)
    full = lambda t: t.expand(n, groups, c * h * ww // groups).reshape(n, c, h, ww)
    ch = lambda t: d(t).view(1, c, 1, 1)
    xhat = ((rows - mean) * rstd).reshape(n, c, h, ww)
    t = xhat * ch(w)
    z = t + ch(b) + (d(r) if r is not None else 0)
    y = _act(z, act)
    sig = torch.sigmoid(z)
    slope = (z > 0).double() if act == 'relu' else sig * (1 + z * (1 - sig)) if act == 'silu' else torch.ones_like(z)
    dz = d(dy) * slope
    a = dz * ch(w)
    m = lambda v: full(v.reshape(n, groups, -1).mean(2, keepdim=True))
    dx = full(rstd) * (a - m(a) - xhat * m(a * xhat))
    s = 24 if act == 'silu' else 0
    mag = (d(dy).abs() * 1.1 if act == 'silu' else dz.abs())
    am = mag * ch(w).abs()
    L = min(n * h * ww, 2048)
    tol = dict(
        y=8 * U * (t.abs() + ch(b).abs() + (d(r).abs() if r is not None else 0)) + (8 * U * (z.abs() + 1) if act == 'silu' else 0),
        dx=full(rstd) * U * ((8 + s) * am + (L + 8 + s) * (m(am) + xhat.abs() * m((am * xhat).abs()))),
        dw=(L + 8 + s) * U * (mag * xhat.abs()).sum((0, 2, 3)), db=(L + 8 + s) * U * mag.sum((0, 2, 3)), dr=(4 + s) * U * mag)
    return dict(y=y, dx=dx, dw=(dz * xhat).sum((0, 2, 3)), db=dz.sum((0, 2, 3)), dr=dz), tol


def _run(x, groups, w, b, r, dy, act, eps=1e-5):
    from alphazero_amd.norm import group_norm_act
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, r)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], eps=eps, act=act, residual=leaves[3])
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    out = dict(y=y.detach(), dx=got[0], dw=got[1], db=got[2])
    if r is not None:
        out['dr'] = got[3]
    with torch.no_grad():
        alone = group_norm_act(x, groups, w, b, eps=eps, act=act, residual=r)
    assert bool(((alone == out['y']) | (alone.isnan() & out['y'].isnan())).all())     # the serving form is the training form
    assert y.is_contiguous(memory_format=torch.channels_last) and y.dtype == x.dtype
    return out


def _check(got, want, tol, dtype, param):
    for k, v in got.items():
        half = HALF[param if k in ('dw', 'db') else dtype]
        tiny = 2.0 ** -25 if (param if k in ('dw', 'db') else dtype) == torch.float16 else 0.0     # half a subnormal step
        assert v.dtype == (param if k in ('dw', 'db') else dtype)
        off = (v.double() - want[k]).abs() - (1 + half) * tol[k] - half * want[k].abs() - tiny
        assert bool((off <= 0).all()), (k, off.max().item(), int((off > 0).sum()))


SHAPES = [(1, 256, 32, 6, 7), (5, 2, 1, 6, 7), (3, 1, 1, 3, 3), (2, 30, 5, 5, 3), (4, 12, 3, 1, 1), (7, 64, 64, 4, 4), (130, 128, 16, 6, 7),
          (2, 1300, 1, 3, 3), (1, 2200, 2, 2, 2), (2, 64, 8, 32, 32), (1, 320, 32, 64, 64), (3, 48, 4, 19, 19), (9, 16, 1, 3, 3),
          (33, 8, 1, 1, 5), (1, 1, 1, 1, 1), (300, 24, 8, 6, 7), (2, 96, 1, 61, 3), (600, 4, 2, 1, 1), (3, 20, 1, 50, 41), (1, 512, 2, 40, 40),
          (2, 6000, 1, 2, 3), (3, 2051, 1, 3, 3), (2, 60, 6, 48, 31), (70, 128, 16, 20, 20)]


@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('dtype,param', [('f32', 'f32'), ('bf16', 'f32'), ('f16', 'f16')])
@pytest.mark.parametrize('act,residual', [('relu', True), ('relu', False), ('silu', True), ('none', True), ('silu', False)])
def test_forward_and_gradients(shape, dtype, param, act, residual):
    n, c, groups, h, w = shape
    dt, pt = DT[dtype], DT[param]
    args = _inputs(n, c, h, w, dt, pt, residual, seed=n * 1000 + c)
    x, wt, b, r, dy = args
    want, tol = _reference(x, groups, wt, b, r, dy, act)
    _check(_run(x, groups, wt, b, r, dy, act), want, tol, dt, pt)


def test_reference_gradients_are_the_differences():
    """The gradients above are the formulas'; here the formulas against differences of y in 64 bits."""
    n, c, groups, h, w = 2, 6, 3, 2, 3
    for act in ('none', 'silu', 'relu'):
        x, wt, b, r, dy = (t.double() for t in _inputs(n, c, h, w, torch.float32, torch.float32, True, 5))
        want, _ = _reference(x, groups, wt, b, r, dy, act)
        loss = lambda *a: (_reference(a[0], groups, a[1], a[2], a[3], dy, act)[0]['y'] * dy).sum().item()
        base = [x, wt, b, r]
        for k, name in enumerate(('dx', 'dw', 'db', 'dr')):
            flat = want[name].contiguous().reshape(-1)
            for i in range(flat.numel()):
                e = torch.zeros(base[k].numel(), dtype=torch.float64, device='cuda')
                e[i] = 1e-6
                e = e.reshape(base[k].shape)
                up, down = (loss(*[t + s * e if j == k else t for j, t in enumerate(base)]) for s in (1, -1))
                # a step of 1e-6: 2e-10 of rounding in each loss over 2e-6, 1e-12 of curvature (no relu passes its border
                # within the step: the inputs are fixed)
                assert abs((up - down) / 2e-6 - flat[i].item()) < 1e-6, (act, name, i)


def test_kernel_gradients_against_differences_of_the_kernel():
    """A step along a random direction, five-point differences of the kernel's own y.  Allowed: the roundings of y over
    the step, what the same differences of the 64-bit formula are off by, and the gradient's own tolerance."""
    n, c, groups, h, w = 3, 32, 4, 6, 7
    x, wt, b, r, dy = _inputs(n, c, h, w, torch.float32, torch.float32, True, 6)
    from alphazero_amd.norm import group_norm_act
    g = torch.Generator().manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g).cuda().contiguous(memory_format=torch.channels_last) if t.dim() == 4
            else torch.randn(t.shape, generator=g).cuda() for t in (x, wt, b, r)]
    got = _run(x, groups, wt, b, r, dy, 'silu')
    want, tol = _reference(x, groups, wt, b, r, dy, 'silu')
    step = 2.0 ** -6
    for k, name in enumerate(('dx', 'dw', 'db', 'dr')):
        def moved(s):
            return [t + s * step * dirs[k] if j == k else t for j, t in enumerate((x, wt, b, r))]
        kernel = lambda s: (lambda a: (group_norm_act(a[0], groups, a[1], a[2], act='silu', residual=a[3]).double() * dy.double()).sum())(moved(s))
        exact = lambda s: (lambda a: (_reference(a[0], groups, a[1], a[2], a[3], dy, 'silu')[0]['y'] * dy.double()).sum())(moved(s))
        five = lambda f: (8 * (f(1) - f(-1)) - (f(2) - f(-2))) / (12 * step)
        analytic = (got[name].double() * dirs[k].double()).sum()
        truth = (want[name] * dirs[k].double()).sum()
        rounding = 1.5 / step * ((tol['y'] + U * want['y'].abs()) * 1.3 * dy.double().abs()).sum()
        allowed = rounding + (five(exact) - truth).abs() + ((tol[name] + U * want[name].abs()) * dirs[k].double().abs()).sum()
        assert (five(kernel) - analytic).abs() <= allowed, (name, (five(kernel) - analytic).item(), allowed.item())


def test_relu_cuts_the_gradient_where_the_sum_passes_zero_in_64_bits():
    """Four million values, a share of them as close to the border as float32 lets them be: the residual is chosen as the
    negated normalised value, so that z is nothing but rounding.  Every sign has to be the exact one."""
    n, c, groups, h, w = 512, 64, 8, 8, 16
    x, wt, b, _, dy = _inputs(n, c, h, w, torch.float32, torch.float32, False, 7)
    full, _ = _reference(x, groups, wt, b, None, dy, 'none')
    r = (-full['y']).float().contiguous(memory_format=torch.channels_last)
    dy = torch.ones_like(dy)
    want, _ = _reference(x, groups, wt, b, r, dy, 'relu')
    got = _run(x, groups, wt, b, r, dy, 'relu')
    assert 0.3 < want['dr'].mean().item() < 0.7
    # the two 64-bit evaluations of z differ by roundings of 2^-53 of terms below 10; a sign may differ within that
    rows = x.double().reshape(n, groups, -1)
    z = full['y'] + r.double()
    sure = z.abs() > 1e-14
    assert torch.equal(got['dr'].double()[sure], want['dr'][sure]) and float(sure.double().mean()) > 0.999


def test_relu_cuts_exactly_in_groups_far_from_zero():
    """Means a thousand spreads away, no bias, no residual: z passes zero where x passes the mean, which lies between two
    float32 values of x."""
    n, c, groups, h, w = 64, 32, 4, 8, 8
    x, wt, _, _, _ = _inputs(n, c, h, w, torch.float32, torch.float32, False, 18, 1000.0, 1e-3)
    b, dy = torch.zeros(c, device='cuda'), torch.ones_like(x)
    want, _ = _reference(x, groups, wt, b, None, dy, 'relu')
    got = _run(x, groups, wt, b, None, dy, 'relu')
    # db counts the open values; the 64-bit mean itself is good to 1e-13 of values 1e-4 apart, so no count may differ
    assert torch.equal(got['db'].double(), want['db'])


def test_constant_groups_have_their_bias():
    """Groups of equal values (an empty board behind a convolution): variance 0, z = bias exactly, relu open where
    bias > 0 and shut where it is 0 or below, no gradient through x."""
    n, c, groups, h, w = 4, 16, 4, 6, 7
    x = torch.full((n, c, h, w), 0.1, device='cuda').contiguous(memory_format=torch.channels_last)
    wt = torch.ones(c, device='cuda')
    b = torch.linspace(-1, 1, c, device='cuda')
    b[3] = 0.0
    got = _run(x, groups, wt, b, None, torch.ones_like(x), 'relu')
    assert torch.equal(got['y'], b.relu().view(1, c, 1, 1).expand(n, c, h, w))
    assert torch.equal(got['db'], (b > 0).float() * n * h * w) and bool((got['dw'].abs() < 1e-5).all())


@pytest.mark.parametrize('offset,gain', [(1e4, 1.0), (-3e3, 1e-1), (0.0, 1e-6), (0.0, 1e6), (0.0, 1e-20)])
def test_large_offsets_and_scales(offset, gain):
    n, c, groups, h, w = 3, 32, 4, 6, 7
    x, wt, b, r, dy = _inputs(n, c, h, w, torch.float32, torch.float32, True, 8, offset, gain)
    want, tol = _reference(x, groups, wt, b, r, dy, 'relu')
    # the statistics' own error: 2^-53 of (mean / spread)^2 in the variance's relative error, some 1e-7 at 3e4
    want_var = max(1.0, (offset / gain if offset else 0.0) ** 2 * 2.0 ** -50 / U)
    _check(_run(x, groups, wt, b, r, dy, 'relu'), want, {k: v * want_var for k, v in tol.items()}, torch.float32, torch.float32)


def test_nan_and_infinity_stay_in_their_group():
    n, c, groups, h, w = 4, 32, 4, 6, 7
    x, wt, b, r, dy = _inputs(n, c, h, w, torch.float32, torch.float32, True, 9)
    clean = _run(x, groups, wt, b, r, dy, 'relu')
    x2 = x.clone(memory_format=torch.preserve_format)
    x2[1, 9, 2, 3] = float('nan')
    x2[2, 20, 0, 0] = float('inf')
    got = _run(x2, groups, wt, b, r, dy, 'relu')
    for k in ('y', 'dx', 'dr'):
        bad = torch.zeros(n, c, h, w, dtype=torch.bool, device='cuda')
        bad[1, 8:16] = bad[2, 16:24] = True
        assert torch.equal(got[k][~bad], clean[k][~bad]), k
    assert bool(got['y'][1, 8:16].isnan().all()) and bool(got['y'][2, 16:24].isnan().all())
    assert bool(got['dx'][1, 8:16].isnan().all())


def test_layouts_strides_and_alignment():
    """The same values in other layouts give the same results: NCHW, a slice of a batch, a slice of channels, storage
    that begins off any 16-byte border, an expanded gradient, two dimensions."""
    from alphazero_amd.norm import group_norm_act
    n, c, groups, h, w = 6, 32, 4, 6, 7
    x, wt, b, r, dy = _inputs(n, c, h, w, torch.float32, torch.float32, True, 10)
    want = _run(x, groups, wt, b, r, dy, 'relu')
    close = lambda a, e: torch.allclose(a, e, rtol=1e-5, atol=1e-5)      # (another width of loads: other orders of sums)

    def odd(t, shift=1):
        buf = torch.empty(t.numel() + 8, dtype=t.dtype, device='cuda')[shift:shift + t.numel()]
        return buf.as_strided(t.shape, t.stride(), buf.storage_offset()).copy_(t)
    for f in (lambda t: t.contiguous(), odd, lambda t: odd(t, 2), lambda t: t.repeat_interleave(2, 0)[::2], lambda t: torch.cat([t, t], 1)[:, :c], lambda t: t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)):
        got = _run(f(x), groups, wt, b, f(r), f(dy), 'relu')
        for k in want:
            assert close(got[k], want[k]), k
    xs = x.detach().requires_grad_()
    group_norm_act(xs, groups, wt, b, act='none').sum().backward()       # an expanded gradient of ones
    ones = _run(x, groups, wt, b, None, torch.ones_like(x), 'none')
    assert torch.equal(xs.grad, ones['dx'])
    flat = _run(x.reshape(n, c * h, w, 1)[:, :, :1], groups, torch.ones(c * h, device='cuda'), torch.zeros(c * h, device='cuda'), None,
                torch.ones(n, c * h, 1, 1, device='cuda'), 'silu')['y']
    two = group_norm_act(x.reshape(n, c * h, w)[:, :, 0], groups, act='silu')
    assert torch.equal(two, flat.reshape(n, c * h))


def test_gradients_of_a_subset():
    from alphazero_amd.norm import group_norm_act
    n, c, groups, h, w = 6, 32, 4, 6, 7
    x, wt, b, r, dy = _inputs(n, c, h, w, torch.float32, torch.float32, True, 11)
    want = _run(x, groups, wt, b, r, dy, 'relu')
    leaves = dict(dx=x, dw=wt, db=b, dr=r)
    for name in leaves:
        t = {k: v.detach().requires_grad_(k == name) for k, v in leaves.items()}
        y = group_norm_act(t['dx'], groups, t['dw'], t['db'], residual=t['dr'])
        (g,) = torch.autograd.grad(y, [t[name]], dy)
        assert torch.equal(g, want[name]), name
    t = x.detach().requires_grad_()
    y = group_norm_act(t, groups, None, None, residual=r)
    ref, tol = _reference(x, groups, torch.ones_like(wt), torch.zeros_like(b), r, dy, 'relu')
    _check(dict(y=y.detach(), dx=torch.autograd.grad(y, [t], dy)[0]), ref, tol, torch.float32, torch.float32)
    # a residual that is also the input, as where a block begins with its norm: the gradients add up
    t = x.detach().requires_grad_()
    y = group_norm_act(t, groups, wt, b, residual=t)
    (g,) = torch.autograd.grad(y, [t], dy)
    both = _run(x, groups, wt, b, x, dy, 'relu')
    assert torch.equal(g, both['dx'] + both['dr'])


def test_same_bits_every_time_and_whatever_the_batch():
    n, c, groups, h, w = 700, 64, 8, 6, 7
    x, wt, b, r, dy = _inputs(n, c, h, w, torch.bfloat16, torch.float32, True, 12)
    first = _run(x, groups, wt, b, r, dy, 'relu')
    for _ in range(3):
        again = _run(x, groups, wt, b, r, dy, 'relu')
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_offsets_beyond_32_bits():
    """More than 2^31 values; the last samples against the same samples alone."""
    n, c, groups, h, w = 8194, 64, 8, 64, 64
    assert n * c * h * w > 2 ** 31
    from alphazero_amd.norm import group_norm_act
    x = torch.zeros(n, h, w, c, dtype=torch.bfloat16, device='cuda').permute(0, 3, 1, 2)
    xs, wt, b, _, dys = _inputs(3, c, h, w, torch.bfloat16, torch.float32, False, 13)
    x[-3:] = xs
    x.requires_grad_()
    wl = wt.detach().requires_grad_()
    y = group_norm_act(x, groups, wl, b, act='silu')
    dy = torch.zeros_like(x, requires_grad=False)
    dy[-3:] = dys
    gx, gw = torch.autograd.grad(y, [x, wl], dy)
    want, tol = _reference(xs, groups, wt, b, None, dys, 'silu')
    _check(dict(y=y[-3:].detach(), dx=gx[-3:], dw=gw), want, tol, torch.bfloat16, torch.float32)
    zero = torch.nn.functional.silu(b).to(torch.bfloat16)
    assert torch.allclose(y[0, :, 0, 0].float(), zero.float(), rtol=2 ** -7) and bool((gx[0] == 0).all())


def test_streams_and_captured_graphs():
    """On a side stream; two captured graphs of forward and backward, replayed in turn with eager work in between."""
    from alphazero_amd.norm import group_norm_act
    n, c, groups, h, w = 40, 64, 8, 6, 7
    sets = [_inputs(n, c, h, w, torch.float32, torch.float32, True, s) for s in (14, 15, 16)]
    want = [_run(x, groups, wt, b, r, dy, 'relu') for x, wt, b, r, dy in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(sets[0][0], groups, *sets[0][1:4], sets[0][4], 'relu')
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[k], want[0][k]) for k in got)
    graphs = []
    for _ in range(2):
        static = [t.clone(memory_format=torch.preserve_format) for t in sets[0]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            leaves = [t.detach().requires_grad_() for t in static[:4]]
            y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], residual=leaves[3])
            grads = torch.autograd.grad(y, leaves, static[4])
        graphs.append((graph, static, dict(zip(('y', 'dx', 'dw', 'db', 'dr'), (y.detach(),) + grads))))
    for turn in range(4):
        for j, (graph, static, out) in enumerate(graphs):
            k = (turn + j) % 3
            for s, t in zip(static, sets[k]):
                s.copy_(t)
            graph.replay()
            eager = _run(sets[k][0], groups, *sets[k][1:4], sets[k][4], 'relu')
            for name in out:
                assert torch.equal(out[name], want[k][name]) and torch.equal(eager[name], want[k][name]), (turn, j, name)
    # both at once, on two streams
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    for j, (graph, static, out) in enumerate(graphs):
        for s, t in zip(static, sets[j]):
            s.copy_(t)
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for j, (_, _, out) in enumerate(graphs):
        assert all(torch.equal(out[name], want[j][name]) for name in out)


def test_second_derivatives_are_refused():
    from alphazero_amd.norm import group_norm_act
    x = torch.randn(2, 8, 3, 3, device='cuda', requires_grad=True)
    (g,) = torch.autograd.grad(group_norm_act(x, 2).square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable|differentiate twice'):
        g.sum().backward()


def test_autocast_keeps_the_convolutions_type():
    from alphazero_amd.models import AlphaZeroC4
    torch.manual_seed(1)
    m = AlphaZeroC4(3, 32, norm='group').cuda()
    x = (torch.rand(16, 2, 6, 7, device='cuda') < 0.2).float()
    valid = torch.ones(16, 7, dtype=torch.bool, device='cuda')
    kinds = []
    m._tower[0]._gn2.register_forward_hook(lambda mod, i, o: kinds.append((o.dtype, o.is_contiguous(memory_format=torch.channels_last))))
    with torch.autocast('cuda', dtype=torch.bfloat16):
        p, v = m(x, valid)
    (p.float().sum() + v.float().sum()).backward()
    assert kinds == [(torch.bfloat16, True)] * 3
    assert all(q.grad is not None and bool(q.grad.isfinite().all()) for q in m.parameters())


def _draws(count):
    import random
    rng = random.Random(2)
    for _ in range(count):
        groups, per = rng.choice([1, 2, 3, 4, 5, 8, 16, 32, 33]), rng.choice([1, 2, 3, 4, 6, 7, 8, 10, 12, 16, 24, 40])
        h, w = rng.choice([(1, 1), (3, 3), (6, 7), (1, 13), (19, 19), (rng.randint(1, 48), rng.randint(1, 48))])
        n = rng.randint(1, max(1, min(700, 400000 // (groups * per * h * w))))
        yield n, groups * per, groups, h, w, rng.choice(list(DT)), rng.choice(['none', 'relu', 'silu']), rng.random() < 0.5, rng.random() < 0.3


@pytest.mark.parametrize('n,c,groups,h,w,dtype,act,residual,off', list(_draws(120)))
def test_drawn_shapes_write_their_own_values_only(n, c, groups, h, w, dtype, act, residual, off):
    """Through the C entry points, outputs in the middle of buffers of a pattern that has to survive (`off`: also one
    value off any 16-byte border), the workspace exactly as large as asked for and between patterns too."""
    import ctypes as C
    from alphazero_amd import _lib
    lib, dt = _lib.load(), DT[dtype]
    x, wt, b, r, dy = _inputs(n, c, h, w, dt, torch.float32, residual, seed=n + c + h)
    g = _lib.GroupNorm(n, h * w, c, groups, ['f32', 'bf16', 'f16'].index(dtype), 0, ['none', 'relu', 'silu'].index(act), 0, 1e-5)
    pad, banks = 4096, []

    def bank(count, kind):
        buf = torch.full((count + 2 * pad + 8,), 7.0, dtype=kind, device='cuda') if kind.is_floating_point else torch.full(
            (count + 2 * pad + 8,), 77, dtype=kind, device='cuda')
        at = pad + (1 if off and kind == dt else 0)
        banks.append((buf, at, count))
        return buf[at:at + count]
    y, dx, dr = (bank(x.numel(), dt) for _ in range(3))
    dw, db = bank(c, torch.float32), bank(c, torch.float32)
    stats = bank(2 * n * groups, torch.float64)
    sizes = [lib.az_group_norm_workspace_bytes(C.byref(g), k) for k in (0, 1)]
    ws = [bank(s, torch.uint8) for s in sizes]
    p = lambda t: None if t is None else t.data_ptr()
    st = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.az_group_norm_act(C.byref(g), p(x), p(wt), p(b), p(r), p(y), p(stats), p(ws[0]) if sizes[0] else None, sizes[0], st))
    _lib.check(lib.az_group_norm_act_backward(C.byref(g), p(dy), p(x), p(wt), p(b), p(r), p(stats), p(dx), p(dw), p(db),
                                              p(dr) if residual else None, p(ws[1]) if sizes[1] else None, sizes[1], st))
    torch.cuda.synchronize()
    for buf, at, count in banks:
        rest = torch.cat([buf[:at], buf[at + count:]])
        assert bool((rest == (7.0 if buf.dtype.is_floating_point else 77)).all()), (buf.dtype, count)
    if not residual:
        assert bool((dr == 7.0).all())
    want, tol = _reference(x, groups, wt, b, r, dy, act)
    cells = lambda t: t.reshape(n, h, w, c).permute(0, 3, 1, 2)
    got = dict(y=cells(y), dx=cells(dx), dw=dw, db=db)
    if residual:
        got['dr'] = cells(dr)
    _check(got, want, tol, dt, torch.float32)


def test_a_graph_kept_and_run_twice_and_inference_mode():
    from alphazero_amd.norm import group_norm_act
    x, wt, b, r, dy = _inputs(9, 24, 6, 7, torch.float32, torch.float32, True, 17)
    leaves = [t.detach().requires_grad_() for t in (x, wt, b, r)]
    y = group_norm_act(leaves[0], 3, leaves[1], leaves[2], residual=leaves[3])
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(p, q) and p.data_ptr() != q.data_ptr() for p, q in zip(first, again))
    with torch.inference_mode():
        assert torch.equal(group_norm_act(x, 3, wt, b, residual=r), y)
    leaves[0].data.add_(0)                                         # (data: no new version)
    y = group_norm_act(leaves[0] * 1, 3, leaves[1], leaves[2])
    with torch.no_grad():
        leaves[1].mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
