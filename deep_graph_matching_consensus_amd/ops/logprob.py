"""Log-probabilities of given matches over a score matrix
(``csrc/hip/match_logprob.hip``): what a matcher answers with - how likely a
given target is, how certain the row is (entropy) and which targets come
next - in one pass over the scores, and the scores' gradient in a second.
The scores are never normalised in memory.  CPU tensors use the oracle in
:mod:`.reference`.
"""
import collections

import torch

from . import _backend
from . import reference as ref

MAX_TOP = 32

MatchLogProbs = collections.namedtuple(
    'MatchLogProbs', ['log_prob', 'entropy', 'top_log_prob', 'top_index'])


def match_log_probs(scores, target, n_cols=None, top=0):
    r"""Row-softmax log-probabilities of given columns, with entropies and
    the best alternatives.

    Args:
        scores (Tensor): ``[rows, columns]`` fp32, bf16 or fp16 scores (not
            normalised); any row stride.  ``-inf`` masks an entry.
        target (Tensor): int64 ``[rows]``; a value outside ``[0, columns)``
            means no given match.
        n_cols (Tensor, optional): int32 ``[rows]`` valid columns of every
            row (the target graph's size); the others count as ``-inf``
            whatever they hold.
        top (int): number of alternatives, at most 32 and the columns.

    Returns a :class:`MatchLogProbs`: ``log_prob [rows]`` (fp32; 0 without a
    given match, ``-inf`` for a masked one), ``entropy [rows]`` (natural
    log; 0 for a row without valid scores), ``top_log_prob [rows, top]`` and
    ``top_index [rows, top]`` (best first, equal scores by column; ``-inf``
    and -1 past a row's valid scores).  Gradients flow from ``log_prob`` and
    ``entropy`` to ``scores``; masked entries get 0, and a masked match (the
    constant ``-inf``) gives none.  A NaN or ``+inf`` score makes its row's
    values NaN (and its alternatives' order is then unspecified).
    """
    if scores.dim() != 2 or scores.size(1) < 1 or \
            not scores.dtype.is_floating_point:
        raise ValueError('scores must be a floating [rows, columns] tensor')
    if target.dtype != torch.long or target.shape != scores.shape[:1] or \
            target.device != scores.device:
        raise ValueError('target must be int64 [rows] on the device of '
                         'scores')
    if n_cols is not None and (
            n_cols.dtype != torch.int32 or n_cols.device != scores.device or
            n_cols.shape != scores.shape[:1]):
        raise ValueError('n_cols must be int32 [rows] on the device of '
                         'scores')
    if not 0 <= int(top) <= min(MAX_TOP, scores.size(1)):
        raise ValueError('top = {} not in 0..{}'.format(
            top, min(MAX_TOP, scores.size(1))))
    if not _backend.use_hip(scores):
        return MatchLogProbs(*ref.match_log_probs(scores, target, n_cols,
                                                  int(top)))
    if scores.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError('match_log_probs takes fp32, bf16 and fp16, got '
                         '{}'.format(scores.dtype))
    if scores.stride(1) != 1 and scores.size(1) > 1:
        scores = scores.contiguous()
    return MatchLogProbs(*_backend.ops().match_logprob.default(
        scores, target.contiguous(),
        None if n_cols is None else n_cols.contiguous(), int(top)))
