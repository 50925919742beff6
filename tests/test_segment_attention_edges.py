"""Segment attention where it can go wrong.

Inputs, the plain form in 64 bits and its element-wise bounds are those of
``test_segment_attention.py``.
"""
import pytest
import torch

from test_segment_attention import _case, _close, _plain, _run


# --------------------------------------------------------------------------
# Sick graphs beside healthy ones whose keys are split
# --------------------------------------------------------------------------
def _sick(st, what, rows, cap=0.0):
    """Rows ``rows`` of ``what`` (graph 0's) hold NaN; everything of the
    other graphs has to be what it is without them."""
    val, tol = _plain(st, cap=cap, half=2 if st['bias'] is not None else 0)
    st[what][rows] = float('nan')
    got = _run(st, 'cuda', cap=cap)
    bad = {n: t for n, t in got.items() if n != 'dbias'}
    nq, nk = int(st['ptr_q'][1]), int(st['ptr_k'][1])
    own = {n: nq if n in ('out', 'dq') else nk for n in bad}
    _close({n: t[own[n]:] for n, t in bad.items()},
           {n: val[n][own[n]:] for n in bad},
           {n: tol[n][own[n]:] for n in bad}, what)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,D', [
    (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64),
    (torch.float32, 128)])
@pytest.mark.parametrize('axes,cap', [(0, 0.0), (1, 2.0)])
@pytest.mark.parametrize('what', ['q', 'k', 'v'])
def test_sick_graph_beside_split_keys(dtype, D, axes, cap, what):
    """Two graphs whose rows share a tile of four waves and whose keys share
    a split; the second one's first key begins no tile of the split."""
    st = _case([200, 200], [3001, 2990], 1, 1, D, dtype, axes=axes, half=2)
    _sick(st, what, slice(198, 200) if what == 'q' else slice(2999, 3001),
          cap)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('what', ['q', 'k', 'v'])
def test_sick_graph_beside_few_rows(dtype, what):
    """New rows of eight graphs in one wave's tile, keys split."""
    st = _case([1, 2, 1, 1, 3, 1, 1, 1],
               [1501, 1403, 1700, 1298, 1499, 1333, 1601, 1477], 2, 1, 64,
               dtype)
    _sick(st, what, slice(0, 1) if what == 'q' else slice(1490, 1501))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_sick_graph_beside_low_scores(dtype):
    """The healthy rows' scores lie near -290: a key that is not there (score
    0) would outweigh all of theirs by more than fp32 holds."""
    st = _case([200, 200], [3001, 2990], 1, 1, 128, dtype)
    st['q'] = (st['q'].float() - 5).to(dtype)
    st['k'] = (st['k'].float() + 5).to(dtype)
    _sick(st, 'v', slice(2999, 3001))
