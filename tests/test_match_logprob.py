"""Log-probabilities of given matches (ops/logprob.py,
csrc/hip/match_logprob.hip) against a plain form in 64 bits.

Tolerances: the arguments of exp and log carry 2^-24 of their size, sums of
V terms at most V steps of 2^-24; gradients are rounded once to the scores'
type.  Alternatives are compared exactly (ties to the lower column).
"""
import math

import pytest
import torch

from deep_graph_matching_consensus_amd.ops import match_log_probs

F = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _case(R, V, dtype, limited=False, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(R, V, generator=g) * scale).to(dtype)
    n = torch.randint(0, V + 1, (R, ), generator=g, dtype=torch.int32) \
        if limited else None
    y = torch.randint(-1, V + 1, (R, ), generator=g)
    return dict(z=z, y=y, n=n, gl=torch.randn(R, generator=g),
                gh=torch.randn(R, generator=g) * 0.3)


def _plain(st, top):
    """Row by row, in 64 bits: values and error bounds."""
    z, V = st['z'].double(), st['z'].size(1)
    R = z.size(0)
    u = torch.finfo(st['z'].dtype).eps / 2
    val = dict(logp=torch.zeros(R).double(), ent=torch.zeros(R).double(),
               lp=torch.full((R, top), -math.inf).double(),
               idx=torch.full((R, top), -1), dz=torch.zeros(R, V).double())
    tol = {k: torch.zeros_like(val[k]) for k in ('logp', 'ent', 'lp', 'dz')}
    for r in range(R):
        nv = V if st['n'] is None else int(st['n'][r])
        y = int(st['y'][r])
        row = z[r, :nv]
        given = 0 <= y < V
        if given:
            val['logp'][r] = -math.inf
        if nv == 0 or not (row > -math.inf).any():
            continue
        live = row > -math.inf
        lse = torch.logsumexp(row, 0)
        lp = row - lse
        p = lp.exp()
        lpf = torch.where(live, lp, torch.zeros_like(lp))
        rowf = torch.where(live, row, torch.zeros_like(row))
        # z - m, m, log of the sum: e on any log-probability
        e = F * ((nv + 8) + 3 * rowf.abs().max() + lpf.abs().max())
        ent = -(p * lpf).sum()
        val['ent'][r] = ent
        tol['ent'][r] = e * (1 + (p * lpf.abs()).sum()) + \
            (nv + 8) * F * ((p * lpf.abs()).sum() + 1)
        if given and y < nv and bool(live[y]):
            val['logp'][r] = lp[y]
            tol['logp'][r] = e + 4 * F * lp[y].abs()
        order = sorted([j for j in range(nv) if bool(live[j])],
                       key=lambda j: (-float(row[j]), j))[:top]
        for q, j in enumerate(order):
            val['idx'][r, q], val['lp'][r, q] = j, lp[j]
            tol['lp'][r, q] = e + 4 * F * lp[j].abs()
        given = given and y < nv and bool(live[y])
        gl = float(st['gl'][r]) if given else 0.0
        gh = float(st['gh'][r])
        dz = -gl * p - gh * p * (lpf + ent)
        ep = p * (e + 2 * F) + 1e-37
        edz = abs(gl) * ep + abs(gh) * (
            ep * (lpf + ent).abs() + p * (e + tol['ent'][r])) + \
            4 * F * (abs(gl) * p + abs(gh) * p * (lpf.abs() + ent))
        if given:
            dz[y] += gl
            edz[y] += 2 * F * abs(gl)
        val['dz'][r, :nv] = dz
        tol['dz'][r, :nv] = edz + u * dz.abs()
        if st['z'].dtype == torch.float16:
            tol['dz'][r, :nv] += 2.0 ** -25     # its subnormal step
    return val, tol


def _run(st, device, top, grad=True):
    z = st['z'].clone().to(device)
    if grad:
        z.requires_grad_(True)
    n = None if st['n'] is None else st['n'].to(device)
    r = match_log_probs(z, st['y'].to(device), n_cols=n, top=top)
    got = dict(logp=r.log_prob, ent=r.entropy, lp=r.top_log_prob,
               idx=r.top_index)
    if grad:
        got['dz'], = torch.autograd.grad(
            [r.log_prob, r.entropy], z,
            [st['gl'].to(device), st['gh'].to(device)])
    return {k: t.detach().cpu() for k, t in got.items()}


def _close(got, val, tol):
    if 'idx' in got:
        assert torch.equal(got['idx'], val['idx'])
    for k, t in got.items():
        if k == 'idx':
            continue
        t, w = t.double(), val[k]
        assert torch.equal(torch.isfinite(t), torch.isfinite(w)), k
        fine = torch.isfinite(w)
        assert (t[~fine] == w[~fine]).all()
        over = (t - w).abs()[fine] - tol[k][fine]
        assert over.numel() == 0 or over.max() <= 0, (k, over.max())


SHAPES = [(1, 1, 1), (3, 5, 3), (40, 19, 3), (17, 16, 16), (5, 33, 32),
          (6, 64, 10), (4, 65, 2), (3, 256, 32), (3, 257, 10), (2, 1001, 5),
          (2, 1024, 0), (3, 2050, 32), (2, 4099, 1)]
LONG = [(2, 8200, 10), (1, 19572, 10), (3, 19993, 7), (2, 33000, 32),
        (1, 70001, 5), (2, 140000, 3)]


@pytest.mark.parametrize('limited', [False, True])
@pytest.mark.parametrize('R,V,top', SHAPES[:9])
def test_oracle_matches_plain_form(R, V, top, limited):
    st = _case(R, V, torch.float32, limited)
    _close(_run(st, 'cpu', top), *_plain(st, top))


def test_gradients_match_differences():
    st = _case(5, 7, torch.float64, True)
    st['n'][:] = torch.tensor([7, 3, 0, 1, 5], dtype=torch.int32)
    # (a masked target's log-probability has no difference quotient)
    st['y'] = torch.tensor([0, 2, -1, 0, 7])
    z = st['z'].requires_grad_(True)
    assert torch.autograd.gradcheck(
        lambda z: match_log_probs(z, st['y'], st['n'])[:2], (z, ))


@pytest.mark.parametrize('kw', [
    dict(scores=torch.zeros(4), target=torch.zeros(4).long()),
    dict(scores=torch.zeros(4, 0), target=torch.zeros(4).long()),
    dict(scores=torch.zeros(4, 3).int(), target=torch.zeros(4).long()),
    dict(scores=torch.zeros(4, 3), target=torch.zeros(3).long()),
    dict(scores=torch.zeros(4, 3), target=torch.zeros(4).int()),
    dict(scores=torch.zeros(4, 3), target=torch.zeros(4).long(), top=4),
    dict(scores=torch.zeros(4, 40), target=torch.zeros(4).long(), top=33),
    dict(scores=torch.zeros(4, 3), target=torch.zeros(4).long(), top=-1),
    dict(scores=torch.zeros(4, 3), target=torch.zeros(4).long(),
         n_cols=torch.zeros(4).long()),
    dict(scores=torch.zeros(4, 3), target=torch.zeros(4).long(),
         n_cols=torch.zeros(3, dtype=torch.int32))])
def test_refusals(kw):
    with pytest.raises(ValueError):
        match_log_probs(**kw)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('limited', [False, True])
@pytest.mark.parametrize('R,V,top', SHAPES)
def test_kernels_match_plain_form(R, V, top, limited, dtype):
    st = _case(R, V, dtype, limited)
    val, tol = _plain(st, top)
    _close(_run(st, 'cuda', top), val, tol)
    _close(_run(st, 'cuda', top, grad=False), val, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('R,V,top', LONG)
def test_long_rows(R, V, top, dtype):
    st = _case(R, V, dtype, limited=R > 1)
    _close(_run(st, 'cuda', top), *_plain(st, top))


@pytest.mark.gpu
@pytest.mark.parametrize('V', [30, 300, 5000, 40000])
def test_equal_scores_go_to_the_lowest_columns(V):
    """All equal, two values only, and -inf among them."""
    for kind in range(3):
        z = torch.zeros(3, V)
        if kind == 1:
            z[:, 1::2] = 1.0
        if kind == 2:
            z[:] = -math.inf
            z[0, V // 2] = 1.0
            z[1, :20] = 2.0
        st = dict(z=z, y=torch.tensor([0, V - 1, 3]), n=None,
                  gl=torch.ones(3), gh=torch.ones(3))
        top = min(V, 32)
        _close(_run(st, 'cuda', top), *_plain(st, top))


@pytest.mark.gpu
@pytest.mark.parametrize('V', [19, 700, 9000])
def test_masked_columns_may_hold_anything(V):
    st = _case(6, V, torch.float32, True)
    st['n'] = torch.tensor([0, 1, V // 2, V, V - 1, 3], dtype=torch.int32)
    val, tol = _plain(st, 3)
    dead = torch.arange(V) >= st['n'].view(-1, 1)
    st['z'][dead] = float('nan')
    st['z'][2, V // 2:] = math.inf
    _close(_run(st, 'cuda', 3), val, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('V', [19, 700, 9000, 70000])
def test_nan_and_inf_scores_make_their_row_nan(V):
    st = _case(3, V, torch.float32)
    st['y'][:] = 0
    st['z'][0, 5], st['z'][2, 7] = float('nan'), math.inf
    got = _run(st, 'cuda', 2)
    for k in ('logp', 'ent'):
        assert torch.isnan(got[k][[0, 2]]).all(), k
        assert torch.isfinite(got[k][1])
    assert torch.isnan(got['dz'][0]).any() and torch.isfinite(
        got['dz'][1]).all()
    assert ((got['idx'] >= -1) & (got['idx'] < V)).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_strided_rows(dtype):
    st = _case(9, 1300, dtype)
    want = _run(st, 'cuda', 4)
    z = st['z'].cuda()
    wide = torch.full((9, 1303), float('nan'), dtype=dtype, device='cuda')
    wide[:, 2:1302] = z
    for view in (wide[:, 2:1302], z.t().contiguous().t()):
        v = view.detach().requires_grad_(True)
        r = match_log_probs(v, st['y'].cuda(), top=4)
        g, = torch.autograd.grad([r.log_prob, r.entropy], v,
                                 [st['gl'].cuda(), st['gh'].cuda()])
        assert torch.equal(r.top_index.cpu(), want['idx'])
        # (other lanes hold the values: the sums' order differs)
        val, tol = _plain(st, 4)
        _close(dict(logp=r.log_prob.detach().cpu(),
                    ent=r.entropy.detach().cpu(),
                    lp=r.top_log_prob.cpu(), idx=r.top_index.cpu(),
                    dz=g.cpu()), val, tol)


@pytest.mark.gpu
def test_one_gradient_only_and_empty_batch():
    st = _case(7, 40, torch.float32)
    for only, zero in (('gl', 'gh'), ('gh', 'gl')):
        part = dict(st)
        part[zero] = torch.zeros(7)
        val, tol = _plain(part, 0)
        z = st['z'].cuda().requires_grad_(True)
        r = match_log_probs(z, st['y'].cuda())
        out = r.log_prob if only == 'gl' else r.entropy
        g, = torch.autograd.grad(out, z, st[only].cuda())
        _close({'dz': g.cpu()}, val, tol)
    z = torch.zeros(0, 5, device='cuda', requires_grad=True)
    r = match_log_probs(z, torch.zeros(0, dtype=torch.long, device='cuda'),
                        top=2)
    r.log_prob.sum().backward()
    assert z.grad.shape == (0, 5) and r.top_index.shape == (0, 2)


@pytest.mark.gpu
@pytest.mark.parametrize('V', [19, 5000, 70000])
def test_repeats_and_captured_replays_are_identical(V):
    st = _case(12, V, torch.float32)
    dev = {k: t.cuda() for k, t in st.items() if t is not None}
    z = dev['z'].requires_grad_(True)

    def step():
        r = match_log_probs(z, dev['y'], top=5)
        g, = torch.autograd.grad([r.log_prob, r.entropy], z,
                                 [dev['gl'], dev['gh']])
        return [t.detach() for t in r] + [g]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        new = _case(12, V, torch.float32, seed=seed)
        with torch.no_grad():
            for k, t in dev.items():
                t.copy_(new[k])
        eager = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    z = torch.randn(3, 16, device='cuda', requires_grad=True)
    y = torch.zeros(3, dtype=torch.long, device='cuda')
    g, = torch.autograd.grad(match_log_probs(z, y).entropy.sum(), z,
                             create_graph=True)
    with pytest.raises(RuntimeError, match='differentiated again'):
        g.sum().backward()
