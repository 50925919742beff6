"""Segment attention where it can go wrong.

Inputs, the plain form in 64 bits and its element-wise bounds are those of
``test_segment_attention.py``.
"""
import math

import pytest
import torch

from deep_graph_matching_consensus_amd.ops import segment_attention
from test_segment_attention import F, _case, _close, _plain, _run


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


# --------------------------------------------------------------------------
# Scores that swallow the log of their own sum
# --------------------------------------------------------------------------
MASKS = [torch.finfo(torch.float32).min, -1e9]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('low', MASKS)
@pytest.mark.parametrize('lq,lk,D,axes', [
    ([6, 40], [6, 40], 32, 1), ([6, 40], [6, 40], 32, 2),
    ([300], [400], 64, 1), ([300], [400], 128, 1),
    ([2, 1], [1300, 700], 64, 1)])
def test_gradients_of_rows_masked_by_a_lowest_value(dtype, low, lq, lk, D,
                                                    axes):
    """Every key masked by a finite value: the row is uniform, and so are its
    gradients.  With q = 0 the scores are the table's alone, so the plain
    form with a table of zeros has the same weights 1 / n and its bounds do
    not grow with the mask."""
    st = _case(lq, lk, 2, 1, D, dtype, axes=axes, half=2)
    st['q'].zero_()
    st['bias'].zero_()
    val, tol = _plain(st, half=2)
    st['bias'].fill_(low)
    got = _run(st, 'cuda')
    _close(got, val, tol, 'q = 0')
    # |q k| < 64: swallowed by a score of -1e9 (a unit of 64 there)
    st['q'] = _case(lq, lk, 2, 1, D, dtype, axes=axes, half=2)['q']
    st['q'] = (st['q'].float() * 0.5).to(dtype)
    z = torch.einsum('ihd,jd->ihj', st['q'].float(), st['k'][:, 0].float())
    assert z.abs().max() * D ** -0.5 * 1.45 < 32
    more = _run(st, 'cuda')
    for n in ('out', 'dq', 'dv', 'dbias'):
        assert torch.equal(more[n], got[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('lq,lk', [([5, 9], [7, 30]), ([200], [300]),
                                   ([2], [1500])])
def test_weights_of_large_equal_scores_sum_to_one(dtype, lq, lk):
    """All keys alike and scores of 2^23, where a unit of fp32 is one: p is 1
    / n, dv the mean of do's columns, to the roundings of 1 / n, the product
    (fp32 steps, bf16 weights) and the output."""
    st = _case(lq, lk, 1, 1, 64, dtype)
    st['q'].fill_(1024.0)
    st['k'].fill_(1024.0)
    got = _run(st, 'cuda')
    u = torch.finfo(dtype).eps / 2
    up = u if dtype == torch.bfloat16 else 0.0
    for b in range(len(lq)):
        sq = slice(*st['ptr_q'][b:b + 2].tolist())
        sk = slice(*st['ptr_k'][b:b + 2].tolist())
        n, m = sk.stop - sk.start, sq.stop - sq.start
        g = st['do'][sq].double()
        want = (g.sum(0, keepdim=True) / n).expand(n, 1, 64)
        tol = (up + (n + m + 16) * F) * g.abs().sum(0, keepdim=True) / n + \
            u * want.abs()
        assert ((got['dv'][sk].double() - want).abs() <= tol).all()


# --------------------------------------------------------------------------
# Bucket layouts and caps at their ends
# --------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('axes', [1, 2])
@pytest.mark.parametrize('lens', [[5, 20], [300]])
def test_one_bucket(dtype, axes, lens):
    """half = 0: one bucket for every offset, whatever its sign."""
    st = _case(lens, None, 2, 2, 32, dtype, axes=axes, half=0)
    assert (st['pos_q'] < 0).any() and (st['pos_q'] > 0).any()
    st['bias'][:] = torch.tensor([[3.0], [-2.0]])
    val, tol = _plain(st, cap=2.0, half=0)
    _close(_run(st, 'cuda', cap=2.0), val, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('cap', [1e3, 1e5, 1e7, 1e9])
@pytest.mark.parametrize('lens', [[5, 20], [300]])
def test_wide_caps(dtype, cap, lens):
    """A cap far above the scores changes nothing: its rounding follows the
    score, not the cap.  Bounds: those of a cap at four times the largest
    score, over the least slope 1 - tanh(1 / 4)^2 that form multiplies by."""
    st = _case(lens, None, 2, 1, 64, dtype, axes=1, half=2)
    z = torch.einsum('ihd,jd->ihj', st['q'].double(), st['k'][:, 0].double())
    near = 4 * float(z.abs().max()) / 8
    assert near < cap
    val, _ = _plain(st, cap=cap, half=2)
    _, tol = _plain(st, cap=near, half=2)
    tol = {n: t / (1 - math.tanh(0.25) ** 2) for n, t in tol.items()}
    _close(_run(st, 'cuda', cap=cap), val, tol)


@pytest.mark.parametrize('kw', [
    dict(cap=1e39), dict(cap=1e-40), dict(cap=1e-20, scale=1e20),
    dict(scale=math.inf), dict(scale=math.nan), dict(scale=1e38),
    dict(scale=-1e39)])
def test_scores_past_fp32_are_refused(kw):
    """A cap or scale that fp32 holds only as 0 or inf makes 0 times inf of
    an ordinary score."""
    q = torch.randn(4, 2, 8)
    p = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError):
        segment_attention(q, q, q, p, **kw)


@pytest.mark.parametrize('device', [
    'cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('cap,scale', [
    (1e30, None), (1e-30, None), (0.0, 1e30), (0.0, -1e30), (0.0, 0.0),
    (2.0, 0.0), (2.0, -0.3)])
def test_caps_and_scales_at_their_ends_are_finite(cap, scale, device):
    q = torch.randn(4, 2, 8, device=device, requires_grad=True)
    p = torch.tensor([0, 4], dtype=torch.int32, device=device)
    out = segment_attention(q, q, q, p, cap=cap, scale=scale)
    g, = torch.autograd.grad(out.square().sum(), q)
    assert torch.isfinite(out).all()
    if abs(scale or 0.0) < 1:       # (else scores of 1e30 have such gradients)
        assert torch.isfinite(g).all()


# --------------------------------------------------------------------------
# Scores past fp32's integers
# --------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('lq,lk,D', [([5, 9], [7, 30], 64), ([200], [300], 64),
                                     ([200], [300], 128), ([2], [1500], 64)])
@pytest.mark.parametrize('axes,scale', [(0, None), (0, -0.125), (1, None)])
def test_scores_of_2_to_the_31(dtype, lq, lk, D, axes, scale):
    """Multiples of 2^31 / sqrt(D) that every type here holds: a row's largest
    scores share its weight, whatever rounds their product with log2(e).

    Bounds: weights 1 / n are exact to the sum's and the division's steps
    (and the type's, where they enter a product in it); <do, v>, <do, o> and
    the sums over rows as in the plain form."""
    st = _case(lq, lk, 2, 1, D, dtype, axes=axes, half=1)
    g = torch.Generator().manual_seed(9)
    st['q'] = (torch.randint(-3, 4, st['q'].shape, generator=g) *
               2.0 ** 17).to(dtype)
    st['k'] = (torch.randint(-3, 4, st['k'].shape, generator=g) *
               2.0 ** 14).to(dtype)
    if axes:
        st['bias'].zero_()
    got = _run(st, 'cuda', scale=scale)
    s = D ** -0.5 if scale is None else scale
    u = torch.finfo(dtype).eps / 2
    up = u if dtype == torch.bfloat16 else 0.0
    for b in range(len(lq)):
        sq = slice(*st['ptr_q'][b:b + 2].tolist())
        sk = slice(*st['ptr_k'][b:b + 2].tolist())
        K, V = st['k'][sk, 0].double(), st['v'][sk, 0].double()
        n, m = K.size(0), sq.stop - sq.start
        dk, dv = torch.zeros_like(K), torch.zeros_like(V)
        edk, edv = torch.zeros_like(K), torch.zeros_like(V)
        for h in range(2):
            Q, G = st['q'][sq, h].double(), st['do'][sq, h].double()
            z = s * Q @ K.t()
            assert z.abs().max() > 2.0 ** 31 / D ** 0.5
            p = torch.softmax(z, dim=-1)
            rp = up + (n + 16) * F
            o, pv = p @ V, p @ V.abs()
            eo = rp * pv + u * o.abs()
            assert ((got['out'][sq, h].double() - o).abs() <= eo).all()
            dp = G @ V.t()
            delta = (G * o).sum(1, keepdim=True)
            edp = (D + 2) * F * G.abs() @ V.abs().t() + \
                (G.abs() * eo).sum(1, keepdim=True) + \
                D * F * (G * o).abs().sum(1, keepdim=True)
            ds = s * p * (dp - delta)
            eds = abs(s) * p * (rp * (dp - delta).abs() + edp) + \
                (up + 4 * F) * ds.abs()
            dq = ds @ K
            edq = eds @ K.abs() + n * F * ds.abs() @ K.abs() + u * dq.abs()
            assert ((got['dq'][sq, h].double() - dq).abs() <= edq).all()
            dk += ds.t() @ Q
            edk += (eds.t() + 2 * m * F * ds.t().abs()) @ Q.abs()
            dv += p.t() @ G
            edv += ((rp + 2 * m * F) * p).t() @ G.abs()
        for t, e, x in ((dk, edk, 'dk'), (dv, edv, 'dv')):
            err = (got[x][sk, 0].double() - t).abs()
            assert (err <= e + u * t.abs()).all(), x


def test_rows_wider_than_a_buffers_range_are_refused():
    """A tile of 128 rows has to lie within 2^31 bytes, whatever its copy."""
    p = torch.zeros(1, dtype=torch.int32)
    q, k = torch.zeros(0, 16416, 128), torch.zeros(0, 513, 128)
    with pytest.raises(ValueError, match='row'):
        segment_attention(q, k, k, p)
    q, k = torch.zeros(0, 16384, 128), torch.zeros(0, 512, 128)
    assert segment_attention(q, k, k, p).shape == q.shape
    # 1 to 8 wide heads take 8 values in a copy
    q = torch.zeros(0, 1 << 18, 3)
    assert segment_attention(q, q, q, p).shape == q.shape
    q = torch.zeros(0, (1 << 18) + 32, 3)
    with pytest.raises(ValueError, match='row'):
        segment_attention(q, q, q, p)
