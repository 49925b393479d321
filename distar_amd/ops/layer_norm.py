"""Layer normalisation with its residual sum, for training and inference.

``layer_norm(x, ...)`` normalises rows; ``add_layer_norm(x, residual, ...)``
first adds a residual and also returns the sum, the stream that a pre-norm
block carries on.  Both take any width, float32, bfloat16 and float16, rows
with a stride, and weights in float32 or the input's type.  Statistics, the
sums over rows of the weight's and bias's gradients, and everything between
load and store are 32-bit; the gradients' sums have a fixed order, so equal
inputs give equal gradients.

On a GPU the kernels in `ops/hip/layer_norm.hip` run; CPU tensors (and
``DISTAR_AMD_DISABLE_HIP=1``) take the eager composition.  Unlike
`ops/residual_ln.py`, which serves the post-norm entity transformer at one
width and type, the statistics are those of the sum as it is stored.
"""
import torch
import torch.nn as nn

from . import hip_ext


def _eager(s, weight, bias, eps):
    dtype = s.dtype
    s = (s.double() if dtype == torch.float64 else s.float()).contiguous()
    d = s - s.mean(-1, keepdim=True)
    y = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(s.dtype)
    if bias is not None:
        y = y + bias.to(s.dtype)
    return y.to(dtype)


def _check(x, weight, bias, eps):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('layer norm needs a last dimension of at least one element')
    if not x.is_floating_point():
        raise TypeError(f'layer norm takes floating point tensors, not {x.dtype}')
    for name, p in (('weight', weight), ('bias', bias)):
        if p is not None and tuple(p.shape) != (x.shape[-1],):
            raise ValueError(f'{name} has shape {tuple(p.shape)}, but rows have '
                             f'{x.shape[-1]} elements')
    if not eps >= 0:
        raise ValueError(f'eps must not be negative, got {eps}')


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    x: (..., C) float32, bfloat16 or float16; weight, bias: (C,) in float32 or
    x's type (both in one), or None.  Returns x's shape and type.
    """
    ext = hip_ext.maybe_ext(x)
    if ext is not None:
        return ext.layer_norm(x, weight, bias, eps)
    _check(x, weight, bias, eps)
    return _eager(x, weight, bias, eps)


def add_layer_norm(x, residual, weight=None, bias=None, eps=1e-5):
    """``s = x + residual`` and ``y = layer_norm(s)``; returns ``(y, s)``.

    residual has x's shape and type; s is stored in that type and normalised as
    stored.  Gradients of both outputs flow to both inputs.
    """
    ext = hip_ext.maybe_ext(x)
    if ext is not None:
        return ext.add_layer_norm(x, residual, weight, bias, eps)
    _check(x, weight, bias, eps)
    if residual.shape != x.shape:
        raise ValueError(f'residual has shape {tuple(residual.shape)}, but x has '
                         f'{tuple(x.shape)}')
    if residual.dtype != x.dtype:
        raise TypeError(f'residual is {residual.dtype}, but x is {x.dtype}')
    s = x + residual
    return _eager(s, weight, bias, eps), s


class FusedLayerNorm(nn.LayerNorm):
    """`nn.LayerNorm` over the last dimension (same state dict) on these
    kernels.  Called with a residual it returns ``(y, x + residual)``."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, **kwargs):
        super().__init__(normalized_shape, eps=eps,
                         elementwise_affine=elementwise_affine, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError('FusedLayerNorm normalises the last dimension only')

    def forward(self, x, residual=None):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f'rows have {x.shape[-1]} elements, not '
                             f'{self.normalized_shape[0]}')
        if residual is None:
            return layer_norm(x, self.weight, self.bias, self.eps)
        return add_layer_norm(x, residual, self.weight, self.bias, self.eps)
