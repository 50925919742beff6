"""The attentional operators under forward-mode autograd, in reference mode, on
large batches."""
import pytest
import torch
from torch.autograd import forward_ad

from deep_graph_matching_consensus_amd.ops import (layer_norm,
                                                   match_log_probs,
                                                   segment_attention)


@pytest.mark.gpu
@pytest.mark.parametrize('which', ['q', 'k', 'v', 'bias'])
def test_attention_refuses_forward_mode(which):
    """A tangent is an error, never dropped."""
    t = dict(q=torch.randn(4, 2, 8), k=torch.randn(4, 2, 8),
             v=torch.randn(4, 2, 8), bias=torch.randn(2, 3))
    t = {n: x.cuda() for n, x in t.items()}
    ptr = torch.tensor([0, 4], dtype=torch.int32, device='cuda')
    pos = torch.arange(4, dtype=torch.int32, device='cuda')
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match='forward'):
            segment_attention(t['q'], t['k'], t['v'], ptr, bias=t['bias'],
                              pos_q=pos)
        with torch.no_grad(), pytest.raises(RuntimeError, match='forward'):
            segment_attention(t['q'], t['k'], t['v'], ptr, bias=t['bias'],
                              pos_q=pos)


@pytest.mark.gpu
@pytest.mark.parametrize('which', ['x', 'residual', 'weight', 'bias'])
def test_norm_refuses_forward_mode(which):
    t = dict(x=torch.randn(4, 8), residual=torch.randn(4, 8),
             weight=torch.randn(8), bias=torch.randn(8))
    t = {n: x.cuda() for n, x in t.items()}
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match='forward'):
            layer_norm(**t)


@pytest.mark.gpu
def test_log_probs_refuse_forward_mode():
    z = torch.randn(4, 9, device='cuda')
    y = torch.zeros(4, dtype=torch.long, device='cuda')
    with forward_ad.dual_level():
        d = forward_ad.make_dual(z, torch.ones_like(z))
        with pytest.raises(RuntimeError, match='forward'):
            match_log_probs(d, y)
