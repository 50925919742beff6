"""Layer norm over the channels of a node batch
(``csrc/hip/layer_norm.hip``): one kernel forward, one backward plus the
fold of the weight gradients' per-workgroup parts (fixed order, no atomics),
with an optional residual added on the way.  CPU tensors use the oracle in
:mod:`.reference`.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _backend
from . import reference as ref

MAX_COLUMNS = 8192


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        grad = any(ctx.needs_input_grad[:4])
        y, s, stat = _backend.ops().layer_norm_fwd(x, residual, weight, bias,
                                                   eps, grad)
        if residual is None:
            s = x
        if grad:
            ctx.save_for_backward(s, weight, stat)
            ctx.set_materialize_grads(False)
        ctx.has_bias = bias is not None
        return (y, s) if residual is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds=None):
        s, weight, stat = ctx.saved_tensors
        if dy is None:
            return ds, ds, None, None, None
        need_w = weight is not None and any(ctx.needs_input_grad[2:4])
        dx, dw, db = _backend.ops().layer_norm_bwd(
            dy.contiguous(), None if ds is None else ds.contiguous(), s,
            stat, weight, need_w)
        return (dx, dx if ctx.needs_input_grad[1] else None,
                dw if need_w else None,
                db if need_w and ctx.has_bias else None, None)


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    r"""``(x - mean) / sqrt(var + eps) * weight + bias`` over the last
    dimension (biased variance, all sums fp32).

    Args:
        x (Tensor): ``[..., C]`` fp32, bf16 or fp16, ``C <= 8192``.
        weight, bias (Tensor, optional): ``[C]``, any floating dtype (fp32
            arithmetic and gradients); ``bias`` needs ``weight``.
        eps (float): variance floor, > 0.
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
    if not eps > 0.0:
        raise ValueError('eps must be > 0')
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
    flat = x.reshape(-1, C).contiguous()
    res = None if residual is None else residual.reshape(-1, C).contiguous()
    weight, bias = (None if t is None else t.float().contiguous()
                    for t in (weight, bias))
    out = _LayerNorm.apply(flat, res, weight, bias, float(eps))
    if residual is None:
        return out.view(x.shape)
    return out[0].view(x.shape), out[1].view(x.shape)
