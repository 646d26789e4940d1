"""Group norm with an activation and a residual sum, channels last (csrc/az_norm.hip): what the networks of
models.AlphaZero(norm='group') put where the reference's have nn.BatchNorm2d + ReLU (alphazero/models.py:6-28).  It keeps
no statistics of the batch, so a network is the same function in training, in self-play and for a single position.

    y = act((x - mean) * rstd * weight + bias + residual)      mean, rstd over a sample's group of channels

On the GPU forward and backward are hand-written kernels behind an autograd function (csrc/az_torch.cpp; no fallback
there: a missing library raises); CPU tensors take the torch statement below."""
import math

import torch
from torch import nn

from . import _lib

ACTS = {'none': 0, 'relu': 1, 'silu': 2}
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _statement(x, num_groups, weight, bias, eps, act, residual):
    """The same function in torch operations, in 64 bits and rounded once."""
    rows = x.double().reshape(x.shape[0], num_groups, math.prod(x.shape[1:]) // num_groups)
    var, mean = torch.var_mean(rows, 2, correction=0, keepdim=True)
    z = ((rows - mean) * torch.rsqrt(var + eps)).reshape(x.shape)
    channel = (1, -1) + (1,) * (x.dim() - 2)
    if weight is not None:
        z = z * weight.double().view(channel)
    if bias is not None:
        z = z + bias.double().view(channel)
    if residual is not None:
        z = z + residual.double()
    if act != 'none':
        z = torch.relu(z) if act == 'relu' else torch.nn.functional.silu(z)
    return z.to(x.dtype)


def _last(t):
    """Channels last, without a copy where it is that already."""
    if t.dim() == 2:
        return t.contiguous()
    return t.contiguous(memory_format=torch.channels_last)


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act='relu', residual=None):
    """act(group_norm(x, num_groups, weight, bias, eps) + residual), channels last.

    x [N, C, H, W] (kept in torch.channels_last; other layouts are copied to it first) or [N, C], float32, bfloat16 or
    float16; residual of x's shape and type; weight and bias [C], both float32 or both of x's type; act 'none', 'relu'
    or 'silu'.  Returns a channels-last tensor of x's type.  Differentiable once with respect to x, weight, bias and
    residual, on the GPU by a backward pass alone: tensors with a forward-mode tangent, torch.func's transforms, batches of
    gradients and tracing (torch.jit.trace, make_fx, torch.export) are refused there.  Statistics are kept in 64 bits and
    the sign of a value next to zero, at which relu cuts the gradient, is decided in them; a group of one value
    (H * W * C / num_groups == 1) has variance 0.  On the GPU values lie below 2^126 and sqrt(var + eps) between 2^-125 and
    2^125."""
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
    return _lib.autograd().group_norm_act(x, weight, bias, residual, num_groups, eps, ACTS[act])


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
