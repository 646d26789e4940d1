"""CPU side of the group norm (alphazero_amd.norm), the group-normalised networks and FlatAdamW: the torch statement
against the formulas, what is refused, and the C entries' checks of their arguments (none of which launches work)."""
import ctypes as C

import numpy as np
import pytest
import torch

from alphazero_amd import _lib
from alphazero_amd.norm import GroupNormAct, group_norm_act


def _formula(x, groups, w, b, eps, act, r):
    """The definition in 64 bits, written with numpy's elementary operations."""
    n, c = x.shape[:2]
    rows = x.reshape(n, groups, -1).astype(np.float64)
    mean = rows.mean(2, keepdims=True)
    var = ((rows - mean) ** 2).mean(2, keepdims=True)
    ch = (1, c) + (1,) * (x.ndim - 2)
    z = ((rows - mean) / np.sqrt(var + eps)).reshape(x.shape) * w.reshape(ch) + b.reshape(ch) + r
    return np.maximum(z, 0) if act == 'relu' else z / (1 + np.exp(-z)) if act == 'silu' else z


@pytest.mark.parametrize('shape,groups', [((3, 8, 6, 7), 4), ((2, 6), 3), ((1, 5, 1, 1), 1), ((4, 2, 3, 3), 1)])
@pytest.mark.parametrize('act', ['none', 'relu', 'silu'])
def test_statement_is_the_formula(shape, groups, act):
    rng = np.random.RandomState(1)
    x, r = rng.randn(*shape).astype(np.float32), rng.randn(*shape).astype(np.float32)
    w, b = rng.rand(shape[1]).astype(np.float32), rng.randn(shape[1]).astype(np.float32)
    y = group_norm_act(*map(torch.from_numpy, (x,)), groups, torch.from_numpy(w), torch.from_numpy(b), act=act,
                       residual=torch.from_numpy(r))
    want = _formula(x, groups, w, b, 1e-5, act, r)
    # a dozen roundings of values of size |z| + 3
    assert np.all(np.abs(y.numpy() - want) <= 16 * 2.0 ** -24 * (np.abs(want) + 6))


def test_module_is_group_norm_with_the_activation_behind_it():
    m, g = GroupNormAct(4, 16), torch.nn.GroupNorm(4, 16)
    assert list(m.state_dict()) == list(g.state_dict())
    x, r = torch.randn(3, 16, 3, 3), torch.randn(3, 16, 3, 3)
    assert torch.allclose(m(x), torch.relu(g(x)), atol=1e-6)
    assert torch.allclose(m(x, r), torch.relu(g(x) + r), atol=1e-6)


def test_an_empty_batch_has_an_empty_result_and_zero_gradients():
    m = GroupNormAct(2, 4)
    x = torch.zeros(0, 4, 3, 3, requires_grad=True)
    m(x).sum().backward()
    assert x.grad.shape == x.shape and torch.equal(m.weight.grad, torch.zeros(4)) and torch.equal(m.bias.grad, torch.zeros(4))


@pytest.mark.parametrize('bad', [
    dict(num_groups=3), dict(num_groups=0), dict(act='gelu'), dict(eps=-1.0), dict(eps=float('nan')), dict(eps=float('inf')),
    dict(x=torch.zeros(2, 8, 3)), dict(weight=torch.ones(7)), dict(weight=torch.ones(8, 1)), dict(bias=torch.ones(8, dtype=torch.float64)),
    dict(residual=torch.zeros(2, 8, 3, 4)), dict(residual=torch.zeros(2, 8, 3, 3, dtype=torch.bfloat16)),
    dict(weight=torch.ones(8, dtype=torch.bfloat16))])
def test_refused_arguments(bad):
    args = dict(x=torch.zeros(2, 8, 3, 3), num_groups=4, weight=None, bias=None)
    args.update(bad)
    with pytest.raises(ValueError):
        group_norm_act(**args)


def test_refused_types():
    with pytest.raises(TypeError):
        group_norm_act(torch.zeros(2, 8, 3, 3, dtype=torch.float64), 4)
    with pytest.raises(ValueError, match='one type'):
        group_norm_act(torch.zeros(2, 8, 3, 3, dtype=torch.bfloat16), 4, torch.ones(8), torch.ones(8, dtype=torch.bfloat16))


def _descriptor(**kw):
    d = dict(batch=2, cells=9, channels=8, groups=4, dtype=0, param_dtype=0, act=1, eps=1e-5)
    d.update(kw)
    g = _lib.GroupNorm()
    for k, v in d.items():
        setattr(g, k, v)
    return g


@pytest.mark.parametrize('bad', [dict(batch=-1), dict(cells=0), dict(channels=0), dict(groups=0), dict(groups=3), dict(dtype=3),
                                 dict(param_dtype=-1), dict(act=3), dict(eps=-1e-5), dict(eps=float('nan')),
                                 dict(cells=1 << 20, channels=1 << 12)])
def test_c_entries_refuse_bad_descriptors(bad):
    lib = _lib.load()
    g = _descriptor(**bad)
    assert lib.az_group_norm_workspace_bytes(C.byref(g), 0) == -1
    p = C.c_void_p(256)
    assert lib.az_group_norm_act(C.byref(g), p, None, None, None, p, None, p, 1 << 40, None) != 0
    assert lib.az_group_norm_act_backward(C.byref(g), p, p, None, None, None, p, p, None, None, None, p, 1 << 40, None) != 0
    assert b'az_group_norm' in lib.az_last_error()


def test_c_entries_refuse_null_pointers_and_small_workspaces():
    lib = _lib.load()
    g, p = _descriptor(), C.c_void_p(256)
    need = lib.az_group_norm_workspace_bytes(C.byref(g), 1)
    assert lib.az_group_norm_act(C.byref(g), None, None, None, None, p, None, p, 1 << 40, None) != 0
    assert lib.az_group_norm_act(C.byref(g), p, None, None, None, None, None, p, 1 << 40, None) != 0
    assert lib.az_group_norm_act_backward(C.byref(g), p, p, None, None, None, None, p, None, None, None, p, 1 << 40, None) != 0
    assert b'null' in lib.az_last_error()
    assert lib.az_group_norm_act_backward(C.byref(g), p, p, None, None, None, p, p, None, None, p, p, 1 << 40, None) != 0
    assert b'without a residual' in lib.az_last_error()
    assert need > 0
    assert lib.az_group_norm_act_backward(C.byref(g), p, p, None, None, None, p, p, p, p, None, p, need - 1, None) != 0
    assert b'workspace' in lib.az_last_error()
    assert lib.az_group_norm_act_backward(C.byref(g), p, p, None, None, None, p, p, p, p, None, C.c_void_p(264), need, None) != 0
    assert b'aligned' in lib.az_last_error()
    assert lib.az_group_norm_workspace_bytes(None, 0) == -1


def test_adamw_c_entries_refuse_bad_arguments():
    lib = _lib.load()
    b = _lib.AdamWBuffers(*([1 << 12] * 10))
    run = lambda **kw: _lib.AdamWRun(**dict(dict(first_block=0, half=0, lr_index=0, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8), **kw))
    call = lambda b, n, runs, bits, **kw: lib.az_adamw_step(
        b, n, (_lib.AdamWRun * max(len(runs), 1))(*runs), len(runs), bits, kw.get('lr_dev'), 0, kw.get('guard'), 0.0, None, None)
    assert call(b, 0, [run()], 32) == 0                            # nothing to do
    for n, runs, bits, kw in [(-1, [run()], 32, {}), (4, [], 32, {}), (4, [run()] * 33, 32, {}), (4, [run()], 16, {}),
                              (4, [run(first_block=1)], 32, {}), (4, [run(), run(first_block=3), run(first_block=2)], 32, {}),
                              (4, [run(), run(first_block=5)], 32, {}), (4, [run(beta1=1.0)], 32, {}), (4, [run(beta2=-0.1)], 32, {}),
                              (4, [run(eps=float('nan'))], 32, {}), (4, [run(lr_index=32)], 32, dict(lr_dev=4096)),
                              (4, [run()], 32, dict(guard=4096))]:
        assert call(b, n, runs, bits, **kw) != 0, (n, bits, kw)
        assert b'az_adamw_step' in lib.az_last_error()
    for k, bits in (('p', 32), ('g', 32), ('m', 32), ('v', 32), ('m8', 8), ('v8', 8), ('top', 8), ('step', 32)):
        short = _lib.AdamWBuffers(*([1 << 12] * 10))
        setattr(short, k, None)
        assert call(short, 4, [run()], bits) != 0 and b'null' in lib.az_last_error(), k
    short = _lib.AdamWBuffers(*([1 << 12] * 10))
    short.g16 = None
    assert call(short, 4, [run(half=1)], 32) != 0 and b'null' in lib.az_last_error()
    odd = _lib.AdamWBuffers(*([1 << 12] * 10))
    odd.m = (1 << 12) + 4
    assert call(odd, 4, [run()], 32) != 0 and b'aligned' in lib.az_last_error()
    assert lib.az_adamw_decode8(None, None, None, 1, None, None, None) != 0
    assert lib.az_adamw_encode8(1 << 12, 1 << 12, 1, 1 << 12, (1 << 12) + 4, 1 << 12, None) != 0


def test_flat_adamw_refuses_what_it_cannot_do():
    from alphazero_amd.optim import FlatAdamW
    p = [torch.nn.Parameter(torch.zeros(3))]
    with pytest.raises(_lib.AzError, match='GPU'):
        FlatAdamW(p)
    for kw in (dict(state_bits=16), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            FlatAdamW(p, **kw)
    with pytest.raises(ValueError, match='requires a gradient'):
        FlatAdamW([torch.nn.Parameter(torch.zeros(3), requires_grad=False)])


@pytest.mark.filterwarnings('ignore:optimizer contains a parameter group with duplicate')
def test_adamw_refuses_a_parameter_twice():
    from alphazero_amd.optim import FlatAdamW
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(ValueError, match='given twice'):
        FlatAdamW([p, torch.nn.Parameter(torch.ones(2)), p])


def test_group_normalised_networks():
    from alphazero_amd.models import AlphaZero, AlphaZeroC4, GroupNormBlock
    from alphazero_amd.net import TTTNetF32, pack_c4_blob_f32, pack_ttt_blob_f32
    from alphazero_amd.train_c4 import supports
    torch.manual_seed(0)
    m = AlphaZeroC4(3, 32, norm='group')
    assert isinstance(m._tower[0], GroupNormBlock) and m._tower[0] is m._tower[2] and m._tower[0]._gn1.num_groups == 4
    assert not any(isinstance(k, torch.nn.BatchNorm2d) for k in m.modules()) and not list(m.buffers())
    assert AlphaZeroC4(1, 12, norm='group')._tower[0]._gn2.num_groups == 1
    assert AlphaZeroC4(1, 12, norm='group', norm_groups=3)._tower[0]._gn2.num_groups == 3
    assert m._tower[0]._c1.weight.is_contiguous(memory_format=torch.channels_last)
    again = AlphaZeroC4(3, 32, norm='group').to(memory_format=torch.contiguous_format)
    again.load_state_dict(m.state_dict())
    x = (torch.rand(5, 2, 6, 7) < 0.2).float()
    valid = torch.ones(5, 7, dtype=torch.bool)
    assert torch.allclose(again(x, valid)[0], m(x, valid)[0], atol=1e-5)
    m.train()
    p, v = m(x, valid)
    m.eval()
    p1, v1 = m(x[2:3], valid[2:3])                                 # training mode, evaluation mode, alone: one function
    assert torch.allclose(p[2:3], p1, atol=1e-5) and torch.allclose(v[2:3], v1, atol=1e-5)
    for kw in (dict(norm='layer'), dict(norm='batch', norm_groups=4)):
        with pytest.raises(ValueError):
            AlphaZeroC4(1, 32, **kw)
    with pytest.raises(ValueError):
        AlphaZeroC4(1, 32, norm='group', norm_groups=5)
    # the kernels that fold batch-norm refuse them
    assert not supports(m)
    with pytest.raises(ValueError, match='batch'):
        pack_c4_blob_f32(m)
    t = AlphaZero((2, 3, 3), (9,), 2, 16, norm='group')
    assert not TTTNetF32.supports(t)
    with pytest.raises(ValueError, match='batch'):
        pack_ttt_blob_f32(t)


def _config(**training):
    from alphazero_amd.config import AlphaZeroConfig
    return AlphaZeroConfig(conf={
        'game': {'module': 'alphazero.games.connectfour', 'name': 'ConnectFour'},
        'model': {'module': 'alphazero.games.connectfour', 'name': 'AlphaZeroC4',
                  'kwargs': {'num_blocks': 1, 'channels_per_block': 8, 'norm': 'group'}},
        'loss': {'module': 'alphazero.loss', 'name': 'AlphaZeroLoss'},
        'training': dict({'num_steps': 10, 'batch_size': 4, 'lr': 1e-3, 'momentum': 0.9, 'weight_decay': 1e-2,
                          'lr_schedule_gamma': 0.1, 'lr_schedule': [5]}, **training)})


def test_training_worker_takes_the_optimizer_from_the_config():
    from alphazero_amd.training import TrainingWorker

    class Window:
        def __len__(self):
            return 0
    tw = TrainingWorker(_config(optimizer='adamw', betas=[0.8, 0.99]), None, Window(), None, 'cpu')
    assert isinstance(tw._optimizer, torch.optim.AdamW) and tw._optimizer.param_groups[0]['betas'] == (0.8, 0.99)
    assert isinstance(TrainingWorker(_config(), None, Window(), None, 'cpu')._optimizer, torch.optim.SGD)
    for bad in (dict(optimizer='lamb'), dict(optimizer='adamw', state_bits=8)):
        with pytest.raises(ValueError):
            TrainingWorker(_config(**bad), None, Window(), None, 'cpu')


def test_autograd_functions_are_bound_to_the_loaded_library():
    m = _lib.autograd()
    assert m is _lib.autograd() and callable(m.group_norm_act)
    with pytest.raises(RuntimeError, match='four entry points'):
        m.bind([])
    assert _lib.autograd() is m
