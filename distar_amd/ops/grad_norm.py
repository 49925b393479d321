"""The norm of a list of gradients together, and clipping to a largest norm.

`grad_norm` and `clip_grad_norm` take float32, bfloat16 and float16 tensors in
any mix, of any sizes and strides, and keep the norm on the device: nothing in
them waits for the GPU.  Sums are 64-bit but for runs of eight, so the norm does
not overflow before it has to.  Their order is fixed by the tensors' sizes and
places in memory: the same tensors give the same norm each time, equal ones in
other places may differ in its last bit.  Replicas that have to agree to the bit
take the norm of one of them, or one bucket laid out alike.
`utils/grad_clip.py` offers them as ``type: global_norm``.

On a GPU the kernels in `ops/hip/grad_norm.hip` run; CPU tensors (and
``DISTAR_AMD_DISABLE_HIP=1``) take the eager composition.
"""
import math

import torch

from . import hip_ext

_ORDERS = {1.0: 1, 2.0: 2, math.inf: 0}


def _prepare(tensors, norm_type):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        raise ValueError('no tensors were given')
    order = _ORDERS.get(float(norm_type))
    if order is None:
        raise ValueError(f'norm_type must be 1, 2 or inf, got {norm_type}')
    return tensors, order


def _check(tensors):
    for t in tensors:
        if not t.is_floating_point() or t.layout != torch.strided:
            raise TypeError(f'gradients must be dense floating point tensors, got '
                            f'{t.dtype}, {t.layout}')
        if t.device != tensors[0].device:
            raise ValueError(f'gradients are on {tensors[0].device} and {t.device}')


def _eager_norm(tensors, order):
    parts = [t.double().abs() for t in tensors if t.numel()]
    if not parts:
        total = torch.zeros((), dtype=torch.float64, device=tensors[0].device)
    elif order == 0:
        total = torch.stack([p.amax() for p in parts]).amax()
    else:
        total = torch.stack([(p * p if order == 2 else p).sum() for p in parts]).sum()
    return (total.sqrt() if order == 2 else total).float()


@torch.no_grad()
def grad_norm(tensors, norm_type=2.0):
    """The norm (1, 2 or inf) over all elements of `tensors`, as a 0-d float32
    tensor on their device."""
    tensors, order = _prepare(tensors, norm_type)
    ext = hip_ext.maybe_ext(tensors[0])
    if ext is not None:
        return ext.clip_grad_norm(tensors, None, order, 0., 0., False)
    _check(tensors)
    return _eager_norm(tensors, order)


@torch.no_grad()
def clip_grad_norm(tensors, max_norm, norm_type=2.0, eps=1e-6, out=None):
    """Scales `tensors` by ``min(1, max_norm / (norm + eps))`` and returns the
    norm before that, as a 0-d float32 tensor on their device.

    In place, or into `out`: a list of tensors of the same shapes in types of
    their own, such as float32 gradients of an optimiser.  Tensors that are
    written must not share memory with each other, nor with others of `tensors`
    (one may be its own output).  A norm of NaN makes the
    results NaN, an infinite one makes them 0 (and infinities NaN), as the
    formula says.
    """
    tensors, order = _prepare(tensors, norm_type)
    if not max_norm >= 0:
        raise ValueError(f'max_norm must not be negative, got {max_norm}')
    if not eps >= 0:
        raise ValueError(f'eps must not be negative, got {eps}')
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(out) != len(tensors):
            raise ValueError(f'out has {len(out)} tensors for {len(tensors)}')
    ext = hip_ext.maybe_ext(tensors[0])
    if ext is not None:
        return ext.clip_grad_norm(tensors, out, order, max_norm, eps, True)
    _check(tensors)
    for o, t in zip(out or [], tensors):
        if o.shape != t.shape:
            raise ValueError(f'an output of shape {tuple(o.shape)} was given for '
                             f'{tuple(t.shape)}')
        if not o.is_floating_point() or o.device != t.device:
            raise TypeError(f'an output is {o.dtype} on {o.device}')
    norm = _eager_norm(tensors, order)
    scale = (max_norm / (norm + eps)).clamp(max=1.0)
    for t, o in zip(tensors, tensors if out is None else out):
        o.copy_(t.to(torch.promote_types(t.dtype, torch.float32)) * scale)
    return norm
