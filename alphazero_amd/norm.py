"""Group norm with an activation and a residual sum, channels last (csrc/az_norm.hip): what the networks of
models.AlphaZero(norm='group') put where the reference's have nn.BatchNorm2d + ReLU (alphazero/models.py:6-28).  It keeps
no statistics of the batch, so a network is the same function in training, in self-play and for a single position.

    y = act((x - mean) * rstd * weight + bias + residual)      mean, rstd over a sample's group of channels

On the GPU forward and backward are hand-written kernels (no fallback there: a missing library raises); CPU tensors
take the torch statement below."""
import ctypes as C
import math
from functools import lru_cache

import torch
from torch import nn

from . import _lib

ACTS = {'none': 0, 'relu': 1, 'silu': 2}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _statement(x, num_groups, weight, bias, eps, act, residual):
    """The same function in torch operations."""
    rows = x.float().reshape(x.shape[0], num_groups, math.prod(x.shape[1:]) // num_groups)
    var, mean = torch.var_mean(rows, 2, correction=0, keepdim=True)
    z = ((rows - mean) * torch.rsqrt(var + eps)).reshape(x.shape)
    channel = (1, -1) + (1,) * (x.dim() - 2)
    if weight is not None:
        z = z * weight.float().view(channel)
    if bias is not None:
        z = z + bias.float().view(channel)
    if residual is not None:
        z = z + residual.float()
    if act != 'none':
        z = torch.relu(z) if act == 'relu' else torch.nn.functional.silu(z)
    return z.to(x.dtype)


@lru_cache(maxsize=4096)
def _descriptor(n, cells, channels, groups, dtype, param_dtype, act, eps):
    """(az_group_norm, forward workspace bytes, backward workspace bytes): functions of the sizes alone."""
    lib = _lib.load()
    g = _lib.GroupNorm(n, cells, channels, groups, dtype, param_dtype, act, 0, eps)
    sizes = [lib.az_group_norm_workspace_bytes(C.byref(g), k) for k in (0, 1)]
    if min(sizes) < 0:
        raise _lib.AzError(lib.az_last_error().decode())
    return (g, *sizes)


def _workspace(nbytes, device):
    # one for each call, from torch's allocator: calls on several streams or in several captured graphs share nothing
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _last(t):
    """Channels last, without a copy where it is that already."""
    if t.dim() == 2:
        return t.contiguous()
    return t.contiguous(memory_format=torch.channels_last)


def _at(t):
    return None if t is None else t.data_ptr()


def _forward(x, num_groups, weight, bias, eps, act, residual, keep):
    """y, the descriptor and (if `keep`) the statistics the backward pass reads; x and residual channels last."""
    cells = x.shape[2] * x.shape[3] if x.dim() == 4 else 1
    param = weight if weight is not None else bias
    d = _descriptor(x.shape[0], cells, x.shape[1], num_groups, DTYPES[x.dtype], 0 if param is None else DTYPES[param.dtype],
                    ACTS[act], eps)
    y = torch.empty_like(x)
    stats = torch.empty(x.shape[0], num_groups, 2, dtype=torch.float64, device=x.device) if keep else None
    ws = _workspace(d[1], x.device)
    _lib.launch(x.device, _lib.load().az_group_norm_act, d[0], x.data_ptr(), _at(weight), _at(bias), _at(residual), y.data_ptr(),
                _at(stats), _at(ws), d[1])
    return y, d, stats


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, num_groups, eps, act):
        y, ctx.descriptor, stats = _forward(x, num_groups, weight, bias, eps, act, residual, True)
        ctx.save_for_backward(x, weight, bias, residual, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, residual, stats = ctx.saved_tensors
        needs = ctx.needs_input_grad
        d = ctx.descriptor
        dy = _last(dy)
        dx = torch.empty_like(x) if needs[0] else None
        dw = torch.empty_like(weight) if needs[1] else None
        db = torch.empty_like(bias) if needs[2] else None
        dr = torch.empty_like(residual) if needs[3] else None
        ws = _workspace(d[2], x.device)
        _lib.launch(x.device, _lib.load().az_group_norm_act_backward, d[0], dy.data_ptr(), x.data_ptr(), _at(weight), _at(bias),
                    _at(residual), stats.data_ptr(), _at(dx), _at(dw), _at(db), _at(dr), _at(ws), d[2])
        return dx, dw, db, dr, None, None, None


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act='relu', residual=None):
    """act(group_norm(x, num_groups, weight, bias, eps) + residual), channels last.

    x [N, C, H, W] (kept in torch.channels_last; other layouts are copied to it first) or [N, C], float32, bfloat16 or
    float16; residual of x's shape and type; weight and bias [C], both float32 or both of x's type; act 'none', 'relu'
    or 'silu'.  Returns a channels-last tensor of x's type.  Differentiable once with respect to x, weight, bias and
    residual.  Statistics are kept in 64 bits and the sign of a value next to zero, at which relu cuts the gradient, is
    decided in them; an empty group of values (H * W * C / num_groups == 1) has variance 0."""
    if act not in ACTS:
        raise ValueError(f"act is 'none', 'relu' or 'silu', got {act!r}")
    if x.dim() not in (2, 4):
        raise ValueError(f'x is [N, C, H, W] or [N, C], got {tuple(x.shape)}')
    if x.dtype not in DTYPES:
        raise TypeError(f'float32, bfloat16 or float16, got {x.dtype}')
    channels, num_groups, eps = x.shape[1], int(num_groups), float(eps)
    if num_groups <= 0 or channels == 0 or channels % num_groups:
        raise ValueError(f'{channels} channels do not divide into {num_groups} groups')
    if not 0.0 <= eps < float('inf'):
        raise ValueError(f'eps must be finite and not negative, got {eps}')
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f'the residual has x\'s shape, type and device: {tuple(x.shape)} {x.dtype} on {x.device}, got '
                         f'{tuple(residual.shape)} {residual.dtype} on {residual.device}')
    for p in (weight, bias):
        if p is not None and (p.shape != (channels,) or p.dtype not in (torch.float32, x.dtype) or p.device != x.device):
            raise ValueError(f'weight and bias are [{channels}], float32 or {x.dtype}, on {x.device}: got {tuple(p.shape)} '
                             f'{p.dtype} on {p.device}')
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f'weight and bias have one type, got {weight.dtype} and {bias.dtype}')
    if not x.is_cuda or x.numel() == 0:
        return _statement(x, num_groups, weight, bias, eps, act, residual)
    x = _last(x)
    residual = None if residual is None else _last(residual)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _GroupNormAct.apply(x, weight, bias, residual, num_groups, eps, act)
    return _forward(x, num_groups, weight, bias, eps, act, residual, False)[0]


class GroupNormAct(nn.GroupNorm):
    """nn.GroupNorm (same parameters, same state_dict) with the activation and an optional residual sum behind it:
    module(x) = act(norm(x)), module(x, r) = act(norm(x) + r)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, act='relu', device=None, dtype=None):
        super().__init__(num_groups, num_channels, eps=eps, affine=affine, device=device, dtype=dtype)
        if act not in ACTS:
            raise ValueError(f"act is 'none', 'relu' or 'silu', got {act!r}")
        self.act = act

    def forward(self, x, residual=None):
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.act, residual)

    def extra_repr(self):
        return super().extra_repr() + f', act={self.act}'
