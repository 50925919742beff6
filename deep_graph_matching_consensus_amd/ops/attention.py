"""Attention inside the segments (graphs) of a packed node batch.

:func:`segment_attention` is the attentional counterpart of the sparse
operators: every node attends to the nodes of its own graph (self-attention,
``ptr_k=None``) or of the paired graph (cross-attention between the source
and target side of a batch of pairs), never across graphs.  Scores may be
capped by ``cap * tanh(z / cap)`` and receive a learned bias by buckets of
the relative position (:func:`bucket_starts`).

On the GPU one HIP kernel per direction walks the keys of each segment with
the running softmax of ``csrc/hip/segment_attention.h``: the score matrix is
never formed, the work list is derived from ``ptr`` on the device (no host
copy; a captured graph may change ``ptr`` and the rows between replays) and
every sum has a fixed order.  fp32 calls on long segments run as "x6" (three
bf16 terms an operand, six products, fp32 sums: ``DGMC_AMD_X6``, as in
:mod:`.gemm`), short ones - and the kernel that sums a table's gradient - on
exact fp32 products.  CPU tensors use the oracle in :mod:`.reference`.
"""
import torch

from . import _backend
from . import gemm
from . import reference as ref

#: Distances from this on share a bucket in any layout.
MAX_DISTANCE = 1 << 22
MAX_GROUP = 32
MAX_DIM = 128
#: Values of one row (heads times the dimension, in eights): the kernels
#: address the 128 rows of a tile within 2^31 bytes of its first.
MAX_ROW = 1 << 21
#: Largest scale and cap, and the smallest cap's reciprocal: fp32 holds what
#: the kernels form of them.
MAX_FACTOR = 1e30
#: Widest cap the bf16 kernels take; their tanh is off by 1e-7 of the cap.
MAX_CAP_BF16 = 64.0


def bucket_starts(half, octave_steps=1):
    """Smallest distance of each of the ``half + 1`` buckets on one side of
    an axis: ``octave_steps`` (1, 2, 4 or 8) buckets of width 1, then as many
    of width 2, 4, ... - the distance 0 is bucket 0 alone."""
    starts, width = [0], 1
    for n in range(half):
        starts.append(starts[-1] + width)
        if (n + 1) % octave_steps == 0:
            width *= 2
    return starts


def bias_width(half, axes=1):
    """Columns of a bias table: ``2 half + 1`` signed buckets per axis."""
    return (2 * half + 1) ** axes


def _check(q, k, v, ptr_q, ptr_k, cap, scale):
    for t, name in ((q, 'q'), (k, 'k'), (v, 'v')):
        if t.dim() != 3:
            raise ValueError('{} must be [nodes, heads, dim], got {}'.format(
                name, tuple(t.shape)))
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError('q, k and v must share dtype and device')
    if not q.dtype.is_floating_point:
        raise ValueError('q, k and v must be floating')
    if k.shape != v.shape or k.size(2) != q.size(2):
        raise ValueError('k and v must agree in shape and with q in the head '
                         'dimension: {} {} {}'.format(
                             tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if not 1 <= q.size(2) <= MAX_DIM:
        raise ValueError('head dimension {} not in 1..{}'.format(
            q.size(2), MAX_DIM))
    if k.size(1) < 1 or q.size(1) < 1 or q.size(1) % k.size(1) or \
            q.size(1) // k.size(1) > MAX_GROUP:
        raise ValueError('{} query heads over {} key heads: need a multiple '
                         'of at most {}'.format(q.size(1), k.size(1),
                                                MAX_GROUP))
    if q.size(1) * (-(-q.size(2) // 8) * 8) > MAX_ROW:
        raise ValueError('{} heads of {} are more than {} values a '
                         'row'.format(q.size(1), q.size(2), MAX_ROW))
    for t in (ptr_q, ptr_k):
        if t.dtype != torch.int32 or t.dim() != 1 or t.numel() < 1 or \
                t.device != q.device:
            raise ValueError('ptr_q / ptr_k must be int32 [segments + 1] on '
                             'the device of q')
    if ptr_q.numel() != ptr_k.numel():
        raise ValueError('ptr_q and ptr_k must name the same segments')
    if ptr_q is ptr_k and q.size(0) != k.size(0):
        raise ValueError('ptr_k=None (self-attention) needs as many keys as '
                         'queries')
    if cap != 0.0 and not 1.0 / MAX_FACTOR <= cap <= MAX_FACTOR:
        raise ValueError('cap must be 0 (none) or within {:g} and {:g}'.format(
            1.0 / MAX_FACTOR, MAX_FACTOR))
    if scale is not None and not abs(scale) <= MAX_FACTOR * min(
            cap or 1.0, 1.0):
        raise ValueError('scale must be at most {:g} in size, of a cap under '
                         '1 that much of it'.format(MAX_FACTOR))


def _check_bias(q, k, bias, pos_q, pos_k, octave_steps):
    """``(pos_q, pos_k, layout)`` of the bias table's buckets."""
    if pos_q is None:
        raise ValueError('bias needs pos_q')
    if pos_k is None:
        if q.size(0) != k.size(0):
            raise ValueError('bias needs pos_k')
        pos_k = pos_q
    pos_q = pos_q.unsqueeze(-1) if pos_q.dim() == 1 else pos_q
    pos_k = pos_k.unsqueeze(-1) if pos_k.dim() == 1 else pos_k
    for p, n in ((pos_q, q.size(0)), (pos_k, k.size(0))):
        if p.dtype != torch.int32 or p.dim() != 2 or p.size(0) != n or \
                p.size(1) not in (1, 2) or p.device != q.device:
            raise ValueError('positions must be int32 [nodes, 1 or 2] on the '
                             'device of q')
    axes = pos_q.size(1)
    if pos_k.size(1) != axes:
        raise ValueError('pos_q and pos_k must have the same axes')
    if bias.dim() != 2 or bias.size(0) != q.size(1) or \
            bias.device != q.device or not bias.dtype.is_floating_point:
        raise ValueError('bias must be a floating [heads, buckets] table on '
                         'the device of q')
    width = bias.size(1) if axes == 1 else \
        int(round(bias.size(1) ** 0.5))
    half = (width - 1) // 2
    if bias_width(half, axes) != bias.size(1) or half > (31, 3)[axes - 1]:
        raise ValueError('{} buckets on {} axes: need (2 half + 1) ** axes '
                         'with half <= {}'.format(bias.size(1), axes,
                                                  (31, 3)[axes - 1]))
    if octave_steps not in (1, 2, 4, 8):
        raise ValueError('octave_steps must be 1, 2, 4 or 8')
    last = bucket_starts(half, octave_steps)[-1]
    if last > MAX_DISTANCE:
        raise ValueError('the last bucket starts at distance {} > {}: fewer '
                         'buckets or more octave_steps'.format(
                             last, MAX_DISTANCE))
    return (pos_q.contiguous(), pos_k.contiguous(),
            (half, octave_steps.bit_length() - 1, float(last)))


def segment_attention(q, k, v, ptr_q, ptr_k=None, scale=None, cap=0.0,
                      bias=None, pos_q=None, pos_k=None, octave_steps=1):
    r"""Softmax attention within segments of packed rows.

    Row ``i`` of segment ``b`` (``ptr_q[b] <= i < ptr_q[b + 1]``) attends to
    the keys ``ptr_k[b] <= j < ptr_k[b + 1]``::

        z_ij = cap * tanh(scale <q_i, k_j> / cap) + bias[h, bucket_ij]
        out_i = sum_j softmax_j(z_ij) v_j

    (``cap=0``: the plain product; ``bias=None``: none).  Rows of segments
    without keys, rows whose scores are all ``-inf`` and rows behind the last
    segment are 0 and pass no gradient; nothing outside a segment's rows is
    read for it, so padding rows may hold anything.

    Args:
        q (Tensor): ``[N_q, heads, dim]`` fp32 or bf16, ``dim <= 128``; any
            node and head strides (e.g. a slice of a joint projection).
        k, v (Tensor): ``[N_k, key_heads, dim]``; ``heads`` is a multiple
            (at most 32) of ``key_heads``: query head ``h`` reads key head
            ``h // (heads // key_heads)``.
        ptr_q, ptr_k (Tensor): int32 ``[segments + 1]``, ascending from 0, on
            the device (``ptr`` of a batch's dense layout).  ``ptr_k=None``:
            the queries' own segments.
        scale (float): default ``dim ** -0.5``.
        cap (float): score cap, 0 for none.  (On the GPU a bf16 call with a
            cap over 64 runs on fp32 copies of ``q``, ``k`` and ``v``, whose
            kernels keep small scores' precision under any cap.)
        bias (Tensor): learned table ``[heads, (2 half + 1) ** axes]`` with
            ``half <= 31`` on one axis, ``half <= 3`` on two; accumulated in
            fp32.  Finite entries below -1e38 count as -1e38.
        pos_q, pos_k (Tensor): int32 ``[N]`` or ``[N, axes]`` node positions
            (clamped to +-2^23); the bucket of a pair on one axis is ``half +-
            b`` where ``b`` is the last entry of :func:`bucket_starts` not
            above ``|pos_k - pos_q|`` and the sign that of the difference.
            Two axes: ``bucket_x * (2 half + 1) + bucket_y``.
        octave_steps (int): buckets per octave of distance.

    Returns ``[N_q, heads, dim]`` in ``q``'s dtype; softmax statistics and
    all sums are fp32.  bf16 products take weights (and in the backward
    scores' gradients) as one bf16 term where the mean segment is long, as two
    where it is short and in a training forward; that rule and the others of
    the work's layout follow the batch's mean segment.  Forward-mode and
    second derivatives are refused.
    """
    if ptr_k is None:
        ptr_k = ptr_q
    _check(q, k, v, ptr_q, ptr_k, cap, scale)
    scale = q.size(2) ** -0.5 if scale is None else float(scale)
    layout = (0, 0, 0.0)
    if bias is not None:
        pos_q, pos_k, layout = _check_bias(q, k, bias, pos_q, pos_k,
                                           octave_steps)
    else:
        pos_q = pos_k = None
    if not _backend.use_hip(q):
        return ref.segment_attention(
            q, k, v, ptr_q, ptr_k, scale, cap, bias, pos_q, pos_k,
            bucket_starts(layout[0], octave_steps))
    dtype = q.dtype
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError('segment_attention takes fp32 and bf16, got '
                         '{}'.format(dtype))
    if dtype == torch.bfloat16 and cap > MAX_CAP_BF16:
        q, k, v = q.float(), k.float(), v.float()
    q, k, v = (t if t.stride(2) == 1 or t.size(2) == 1 else t.contiguous()
               for t in (q, k, v))
    if bias is not None:
        bias = bias.float().contiguous()
    return _backend.ops().segment_attention.default(
        q, k, v, bias, ptr_q.contiguous(), ptr_k.contiguous(), pos_q, pos_k,
        scale, float(cap), *layout, gemm.NT_X6).to(dtype)
