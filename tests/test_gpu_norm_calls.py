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
