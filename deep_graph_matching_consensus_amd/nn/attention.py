"""Attention layer over packed graph batches.

:class:`AttentionConv` stands beside the message-passing layers where the
neighbourhood is the whole graph: every node attends to all nodes of its own
graph, or to those of the paired graph (``other=``), with a learned bias by
buckets of the nodes' relative position in place of an edge list.
"""
import torch
from torch.nn import Linear, Parameter

from ..graph.dense import dense_layout
from ..ops.attention import bias_width, segment_attention
from ..ops.gemm import linear
from ..ops.norm import layer_norm


class AttentionConv(torch.nn.Module):
    r"""``x + W_o attend(norm(x))`` over the graphs of a batch.

    Args:
        channels (int): feature size (kept by the layer).
        heads (int): query heads, ``channels / heads`` each (at most 128).
        key_heads (int, optional): key / value heads shared by the query
            heads (default: ``heads``).
        cap (float): score cap ``cap * tanh(z / cap)``, 0 for none.
        axes (int): position axes of the bias (0: no bias, 1 or 2).
        half (int): signed buckets per axis, ``2 half + 1``.
        octave_steps (int): buckets per octave of distance.
        eps (float): of the norm.

    Without a position bias it is an encoder of :class:`~..models.DGMC`, which
    calls it with the graphs' ``batch`` vector in place of their edges.
    """

    takes_batch = True

    def __init__(self, channels, heads, key_heads=None, cap=0.0, axes=0,
                 half=3, octave_steps=1, eps=1e-5):
        super(AttentionConv, self).__init__()
        key_heads = heads if key_heads is None else key_heads
        assert channels % heads == 0 and heads % key_heads == 0
        assert axes in (0, 1, 2)
        self.channels, self.heads, self.key_heads = channels, heads, key_heads
        self.in_channels = self.out_channels = channels
        self.dim = channels // heads
        self.cap, self.axes, self.eps = cap, axes, eps
        self.octave_steps = octave_steps
        self.norm_weight = Parameter(torch.ones(channels))
        self.norm_bias = Parameter(torch.zeros(channels))
        self.query = Linear(channels, channels)
        self.key_value = Linear(channels, 2 * key_heads * self.dim)
        self.out = Linear(channels, channels)
        if axes:
            self.table = Parameter(torch.zeros(heads,
                                               bias_width(half, axes)))
        else:
            self.register_parameter('table', None)

    def reset_parameters(self):
        self.norm_weight.data.fill_(1.0)
        self.norm_bias.data.fill_(0.0)
        for lin in (self.query, self.key_value, self.out):
            lin.reset_parameters()
        if self.table is not None:
            self.table.data.fill_(0.0)

    def forward(self, x, batch=None, pos=None, other=None):
        r"""``x [sum N, channels]`` with its ``batch`` vector (``None``: one
        graph) and, for a layer with a bias, int32 positions ``pos [sum N,
        axes]``; ``other = (x_o, batch_o, pos_o)``: the paired graphs to
        attend to (``x``'s own otherwise)."""
        if self.axes:
            for p in (pos, ) if other is None else (pos, other[2]):
                axes = 0 if p is None else 1 if p.dim() == 1 else p.size(-1)
                if axes != self.axes:
                    raise ValueError('{} needs positions pos [nodes, '
                                     '{}]'.format(self, self.axes))
        ptr = dense_layout(batch, x.size(0), x.device).ptr
        h = layer_norm(x, self.norm_weight, self.norm_bias, self.eps)
        q = linear(h, self.query.weight, self.query.bias)
        ptr_o, pos_o, h_o = None, pos, h
        if other is not None:
            x_o, batch_o, pos_o = other
            ptr_o = dense_layout(batch_o, x_o.size(0), x_o.device).ptr
            h_o = layer_norm(x_o, self.norm_weight, self.norm_bias, self.eps)
        kv = linear(h_o, self.key_value.weight, self.key_value.bias)
        kv = kv.view(-1, 2 * self.key_heads, self.dim)
        o = segment_attention(
            q.view(-1, self.heads, self.dim), kv[:, :self.key_heads],
            kv[:, self.key_heads:], ptr, ptr_o, cap=self.cap,
            bias=self.table, pos_q=pos if self.axes else None,
            pos_k=pos_o if self.axes else None,
            octave_steps=self.octave_steps)
        o = linear(o.reshape(-1, self.channels), self.out.weight,
                   self.out.bias)
        return x + o.to(x.dtype)

    def __repr__(self):
        return '{}({}, heads={}, key_heads={}, cap={}, axes={})'.format(
            self.__class__.__name__, self.channels, self.heads,
            self.key_heads, self.cap, self.axes)


__all__ = ['AttentionConv']
