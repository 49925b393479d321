"""Linear layers with bias, activation and residual in one kernel.

``linear_act(x, weight, bias, activation, residual)`` computes
``act(x W^T + b) + residual`` on the matrix cores with 32-bit sums, rounded once
when it is stored, and has a backward pass of its own.  bfloat16 and float16;
weights and biases may be float32 masters, then the weight is cast for the call
and both gradients come in float32.  `ops/linear_relu.py` offers the relu
through the library's product.

On a GPU the kernels in `ops/hip/linear_act.hip` run; CPU tensors (and
``DISTAR_AMD_DISABLE_HIP=1``) take the eager composition.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import hip_ext

ACTIVATIONS = {None: 0, 'relu': 1, 'gelu': 2, 'silu': 3}


def _autocasts(x):
    kind = x.device.type
    return torch.amp.is_autocast_available(kind) and torch.is_autocast_enabled(kind)


def _eager(x, weight, bias, activation, residual):
    wide = torch.promote_types(x.dtype, torch.float32)
    z = x.to(wide) @ weight.to(x.dtype).to(wide).t()
    if bias is not None:
        z = z + bias.to(wide)
    if activation == 'relu':
        z = F.relu(z)
    elif activation == 'gelu':
        z = F.gelu(z)
    elif activation == 'silu':
        z = F.silu(z)
    if residual is not None:
        z = z + residual.to(wide)
    return z.to(x.dtype)


def linear_act(x, weight, bias=None, activation=None, residual=None):
    """``act(x @ weight.T + bias) + residual``.

    x: (..., K) bfloat16 or float16; weight: (N, K) and bias: (N,), or None, in
    x's type or float32; residual: (..., N) in x's type, or None.
    activation: None, 'relu', 'gelu' (by the error function) or 'silu'.
    Returns (..., N) in x's type.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f'activation must be one of {list(ACTIVATIONS)}, got '
                         f'{activation!r}')
    ext = hip_ext.maybe_ext(x)
    if ext is not None:
        return ext.linear_act(x, weight, bias, residual, ACTIVATIONS[activation])
    return _composition(x, weight, bias, activation, residual)


def _composition(x, weight, bias, activation, residual):
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f'x of shape {tuple(x.shape)} does not fit a weight of shape '
                         f'{tuple(weight.shape)}')
    if weight.numel() == 0:
        raise ValueError('weight is empty')
    if not x.is_floating_point():
        raise TypeError(f'x must be floating point, not {x.dtype}')
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f'bias has shape {tuple(bias.shape)} for {weight.shape[0]} outputs')
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None and t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f'{name} is {t.dtype}, but x is {x.dtype}')
    if residual is not None:
        if residual.shape != (*x.shape[:-1], weight.shape[0]):
            raise ValueError(f'residual has shape {tuple(residual.shape)} for an output of '
                             f'{(*x.shape[:-1], weight.shape[0])}')
        if residual.dtype != x.dtype:
            raise TypeError(f'residual is {residual.dtype}, but x is {x.dtype}')
    if not _autocasts(x):
        return _eager(x, weight, bias, activation, residual)
    # autocast would take the product's sums out of 32 bits
    with torch.autocast(x.device.type, enabled=False):
        return _eager(x, weight, bias, activation, residual)


class LinearAct(nn.Linear):
    """`nn.Linear` (same state dict) with an activation and, when called with
    one, a residual in the epilogue.  Under autocast it runs in autocast's type.
    The kernels take bfloat16 and float16; float32 on a GPU, as a model without
    autocast has it, goes through torch's float32 product as in `nn.Linear`."""

    def __init__(self, in_features, out_features, bias=True, activation=None, **kwargs):
        super().__init__(in_features, out_features, bias=bias, **kwargs)
        if activation not in ACTIVATIONS:
            raise ValueError(f'activation must be one of {list(ACTIVATIONS)}, got '
                             f'{activation!r}')
        self.activation = activation

    def forward(self, x, residual=None):
        if _autocasts(x):
            dtype = torch.get_autocast_dtype(x.device.type)
            x = x.to(dtype)
            residual = None if residual is None else residual.to(dtype)
        if x.is_cuda and x.dtype == torch.float32:
            return _composition(x, self.weight, self.bias, self.activation, residual)
        return linear_act(x, self.weight, self.bias, self.activation, residual)
