"""What the group norm's GPU entry refuses before it touches memory, asked with CPU tensors where no GPU is needed for it;
and its kernels' limits, through C entries that launch nothing."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from alphazero_amd import _lib
from alphazero_amd.norm import group_norm_act


def _entry(x, w=None, b=None, r=None):
    return _lib.autograd().group_norm_act(x, w, b, r, 2, 1e-5, 1)


@pytest.mark.parametrize('which', ['x', 'w', 'b', 'r'])
@pytest.mark.parametrize('grad', [False, True])
def test_forward_mode_tangents_are_refused(which, grad):
    """A dual tensor: its tangent would be lost in the kernel.  (The CPU statement has the derivative.)"""
    t = dict(x=torch.randn(2, 4, 3, 3), w=torch.ones(4), b=torch.zeros(4), r=torch.randn(2, 4, 3, 3))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            _entry(**t)
        y = group_norm_act(t['x'], 2, t['w'], t['b'], residual=t['r'])
        assert forward_ad.unpack_dual(y).tangent is not None


def test_functorch_transforms_are_refused():
    x = torch.randn(2, 4, 3, 3)
    for call in (lambda: torch.func.vmap(lambda t: _entry(t))(x[None]), lambda: torch.func.grad(lambda t: _entry(t).sum())(x),
                 lambda: torch.func.jvp(_entry, (x,), (x,)), lambda: torch.func.vmap(lambda t: _entry(x, t))(torch.ones(3, 4))):
        with pytest.raises(NotImplementedError, match='group_norm_act'):
            call()


def test_tracing_is_refused():
    """A trace would hold the result's allocation alone.  (The CPU statement is traced as ever.)"""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch._subclasses.fake_tensor import FakeTensorMode
    x = torch.randn(2, 4, 3, 3)
    for leaf in (x, x.clone().requires_grad_()):
        with pytest.raises(NotImplementedError, match='traced'):
            torch.jit.trace(_entry, (leaf,), check_trace=False)
        for mode in ('real', 'fake', 'symbolic'):
            with pytest.raises(NotImplementedError, match='traced'):
                make_fx(lambda t: _entry(t), tracing_mode=mode)(leaf)
            with pytest.raises(NotImplementedError, match='traced'):
                make_fx(lambda t: _entry(t), tracing_mode=mode, pre_dispatch=True)(leaf)
    with FakeTensorMode():
        fake = torch.empty(2, 4, 3, 3)
        with pytest.raises(NotImplementedError, match='traced'):
            _entry(fake)
    with pytest.raises(NotImplementedError, match='memory of their own'):
        _entry(fake)
    traced = torch.jit.trace(lambda t: group_norm_act(t, 2), (x,), check_trace=False)
    again = torch.randn(2, 4, 3, 3)
    assert torch.equal(traced(again), group_norm_act(again, 2))


def _descriptor(**kw):
    g = _lib.GroupNorm()
    for k, v in dict(dict(batch=1, cells=9, channels=8, groups=4, act=1, eps=1e-5), **kw).items():
        setattr(g, k, v)
    return g


def _workspace(backward, **kw):
    import ctypes as C
    return _lib.load().az_group_norm_workspace_bytes(C.byref(_descriptor(**kw)), backward)


@pytest.mark.parametrize('cells', [46340 ** 2, 2 ** 31 - 1, 2 ** 31 - 31])
@pytest.mark.parametrize('dtype', [0, 1])
def test_workspace_of_the_longest_samples(cells, dtype):
    """One channel, samples up to the limit of 2^31 - 1 values: 16 bytes of partial sums for each of at least two and at most
    one chunk of 256 rows, and 8 for each in the backward pass."""
    forward, backward = (_workspace(k, cells=cells, channels=1, groups=1, dtype=dtype) for k in (0, 1))
    assert forward % 16 == 0 and 2 <= forward // 16 <= cells // 256 and backward == forward // 16 * 24


@pytest.mark.skipif(torch.cuda.is_available(), reason='asked where nothing could be launched')
@pytest.mark.parametrize('big', [
    dict(batch=2 ** 26, cells=1, channels=48, groups=16),                     # one channel a thread, held in registers
    dict(batch=2 ** 26, cells=42, channels=128, groups=16),                   # the same, several
    dict(batch=2 ** 24, cells=361, channels=512, groups=2),                   # teams of 1024
    dict(batch=2 ** 22, cells=4096, channels=1024, groups=32),                # two passes
    dict(batch=2 ** 31 - 1, cells=1, channels=64, groups=64)])
def test_launches_of_too_many_work_items_are_refused(big):
    """Before the first launch: no pointer here is one."""
    import ctypes as C
    lib, p = _lib.load(), C.c_void_p(256)
    g = _descriptor(**big)
    assert lib.az_group_norm_act(C.byref(g), p, None, None, None, p, None, p, 1 << 60, None) != 0
    assert b'work-items' in lib.az_last_error()
    if big['cells'] == 4096:
        assert lib.az_group_norm_act_backward(C.byref(g), p, p, None, None, None, p, p, p, p, None, p, 1 << 60, None) != 0
        assert b'work-items' in lib.az_last_error()


@pytest.mark.parametrize('case', [dict(batch=2 ** 24, cells=42, channels=256, groups=32), dict(batch=2 ** 23, cells=361, channels=192, groups=16, dtype=1),
                                  dict(batch=1, cells=2 ** 20, channels=255, groups=1), dict(batch=1, cells=2 ** 23, channels=255, groups=1, dtype=2)])
def test_parameter_gradients_are_added_in_chains_of_2048_rows(case):
    """What that takes at the least: a workgroup of at most 1024 threads that hold 16 bytes of a row each, and add 2048 of them
    up, ends in one row of partial sums for its channels."""
    size = 4 if case.get('dtype', 0) == 0 else 2
    rows = _workspace(1, **case) // (8 * case['channels'])
    one = 1024 * 2048 * (16 // size) // case['channels']
    if case['batch'] == 1:
        one = 2048 * 256 // 255                    # (an odd number of channels: one to a thread, 256 threads)
    assert rows >= case['batch'] * case['cells'] // one


@pytest.mark.parametrize('offset', [0.0, 1e4, 1e6])
@pytest.mark.parametrize('act', ['none', 'relu', 'silu'])
def test_the_cpu_statement_keeps_its_statistics_in_64_bits_too(offset, act):
    """y and the gradients of x, weight, bias and residual against the same formulas on 64-bit inputs: one rounding of each, and
    what two 64-bit means of `offset` are apart (2^-52 of it), by rstd |w| < 2, for each term."""
    n, c, groups, h, w = 5, 12, 3, 6, 7
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g)
    x, wt, b, r, dy = rnd(n, c, h, w) + offset, 1 + 0.3 * rnd(c), 0.3 * rnd(c), rnd(n, c, h, w), rnd(n, c, h, w)
    leaves = [t.clone().requires_grad_() for t in (x, wt, b, r)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], act=act, residual=leaves[3])
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    exact = [t.double().requires_grad_() for t in (x, wt, b, r)]
    rows = exact[0].reshape(n, groups, -1)
    centred = rows - rows.mean(2, keepdim=True)
    z = (centred / torch.sqrt((centred ** 2).mean(2, keepdim=True) + 1e-5)).reshape(x.shape) * exact[1].view(1, c, 1, 1)
    z = z + exact[2].view(1, c, 1, 1) + exact[3]
    want_y = {'none': lambda t: t, 'relu': torch.relu, 'silu': torch.nn.functional.silu}[act](z)
    want = [want_y.detach(), *torch.autograd.grad(want_y, exact, dy.double())]
    for k, (a, e) in enumerate(zip(got, want)):
        terms = n * h * w if k in (2, 3) else 4
        assert bool(((a.double() - e).abs() <= 2.0 ** -24 * (1.01 * e.abs() + 1e-6) + terms * offset * 2.0 ** -51).all()), k
