"""Layer norm over the channels of a node batch
(``csrc/hip/layer_norm.hip``): one kernel forward, one backward plus the
fold of the weight gradients' per-workgroup parts (fixed order, no atomics),
with an optional residual added on the way.  CPU tensors use the oracle in
:mod:`.reference`.
"""
import torch

from . import _backend
from . import reference as ref

MAX_COLUMNS = 8192


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    r"""``(x - mean) / sqrt(var + eps) * weight + bias`` over the last
    dimension (biased variance, all sums fp32).

    Args:
        x (Tensor): ``[..., C]`` fp32, bf16 or fp16, ``C <= 8192``.
        weight, bias (Tensor, optional): ``[C]``, any floating dtype (fp32
            arithmetic and gradients); ``bias`` needs ``weight``.
        eps (float): variance floor, > 0 in fp32.
        residual (Tensor, optional): like ``x``; the norm is then of ``s = x
            + residual`` (in ``x``'s dtype) and ``(y, s)`` is returned.

    Returns ``y`` (``(y, s)`` with ``residual``) in ``x``'s dtype.
    """
    if x.dim() < 1 or not x.dtype.is_floating_point:
        raise ValueError('x must be a floating [..., C] tensor')
    C = x.size(-1)
    if not 1 <= C <= MAX_COLUMNS:
        raise ValueError('{} columns not in 1..{}'.format(C, MAX_COLUMNS))
    for t, name in ((weight, 'weight'), (bias, 'bias')):
        if t is not None and (t.shape != (C, ) or t.device != x.device or
                              not t.dtype.is_floating_point):
            raise ValueError('{} must be floating [{}] on the device of '
                             'x'.format(name, C))
    if bias is not None and weight is None:
        raise ValueError('bias needs weight')
    if not torch.finfo(ref.sum_dtype(x.dtype)).tiny <= eps < float('inf'):
        raise ValueError('eps must be finite, > 0 and a normal number of '
                         'fp32')
    if residual is not None and (residual.shape != x.shape or
                                 residual.dtype != x.dtype or
                                 residual.device != x.device):
        raise ValueError('residual must have the shape, dtype and device of '
                         'x')
    if not _backend.use_hip(x):
        return ref.layer_norm(x, weight, bias, eps, residual)
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError('layer_norm takes fp32, bf16 and fp16, got '
                         '{}'.format(x.dtype))
    weight, bias = (None if t is None else t.float().contiguous()
                    for t in (weight, bias))
    out = _backend.ops().layer_norm.default(x, residual, weight, bias,
                                            float(eps))
    return out[0] if residual is None else tuple(out)
