"""Attention inside the segments of a packed batch (ops/attention.py,
csrc/hip/segment_attention*) against a plain dense form in 64 bits.

Tolerances follow from the arithmetic (``_plain`` carries them element by
element): every product and sum is fp32 (2^-24 a step, at most as many steps
as terms), P, dS and the outputs are rounded to the input type (bf16: 2^-8
relative each), and the errors are carried through the formulas.
"""
import math

import pytest
import torch

from deep_graph_matching_consensus_amd.ops import segment_attention
from deep_graph_matching_consensus_amd.ops import reference as ref
from deep_graph_matching_consensus_amd.ops.attention import (bias_width,
                                                             bucket_starts)

F = 2.0 ** -24


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _ptr(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)),
                        dtype=torch.int32)


def _plain_bucket(d, half, steps):
    """Signed bucket of one offset, by walking the buckets' widths."""
    b, start = 0, 1                  # bucket 0 is the distance 0 alone
    while b < half and abs(int(d)) >= start:
        b += 1
        start += 2 ** (b // steps)
    return half + (b if d > 0 else -b)


def _inputs(lq, lk, H, KV, D, dtype, axes=0, half=0, seed=0, scale=1.0,
            tail=0, span=12):
    g = torch.Generator().manual_seed(seed)

    def rnd(*shape):
        return (torch.randn(shape, generator=g) * scale).to(dtype)

    nq, nk = sum(lq) + tail, sum(lk) + tail
    st = dict(q=rnd(nq, H, D), k=rnd(nk, KV, D), v=rnd(nk, KV, D),
              do=rnd(nq, H, D), ptr_q=_ptr(lq), ptr_k=_ptr(lk), bias=None,
              pos_q=None, pos_k=None)
    if axes:
        st['bias'] = (torch.randn(H, bias_width(half, axes), generator=g) *
                      0.7)
        st['pos_q'] = torch.randint(-span, span, (nq, axes), generator=g,
                                    dtype=torch.int32)
        st['pos_k'] = torch.randint(-span, span, (nk, axes), generator=g,
                                    dtype=torch.int32)
    return st


def _plain(st, cap=0.0, scale=None, half=0, steps=1):
    """Values and error bounds, head by head and segment by segment."""
    q, k, v, do = (st[n].double() for n in ('q', 'k', 'v', 'do'))
    H, KV, D = q.size(1), k.size(1), q.size(2)
    scale = D ** -0.5 if scale is None else scale
    u = _u(st['q'].dtype)
    up = u if st['q'].dtype == torch.bfloat16 else 0.0
    val = {n: torch.zeros_like(t) for n, t in
           (('out', q), ('dq', q), ('dk', k), ('dv', v))}
    tol = {n: torch.zeros_like(t) for n, t in val.items()}
    if st['bias'] is not None:
        T = st['bias'].double()
        val['dbias'], tol['dbias'] = torch.zeros_like(T), torch.zeros_like(T)
    pq, pk = st['ptr_q'].tolist(), st['ptr_k'].tolist()
    for b in range(len(pq) - 1):
        sq, sk = slice(pq[b], pq[b + 1]), slice(pk[b], pk[b + 1])
        if sq.start == sq.stop or sk.start == sk.stop:
            continue
        n = sk.stop - sk.start
        m = sq.stop - sq.start
        if st['bias'] is not None:
            side = 2 * half + 1
            idx = torch.zeros(m, n, dtype=torch.long)
            for x in range(st['pos_q'].size(1)):
                lim = 2 ** 23        # positions are clamped to this
                d = st['pos_k'][sk, x].long().clamp(-lim, lim)[None] - \
                    st['pos_q'][sq, x].long().clamp(-lim, lim)[:, None]
                idx = idx * side + torch.tensor(
                    [[_plain_bucket(e, half, steps) for e in r]
                     for r in d.tolist()]).view(m, n)
        for h in range(H):
            g = h // (H // KV)
            Q, K, V, G = q[sq, h], k[sk, g], v[sk, g], do[sq, h]
            s = scale * Q @ K.t()
            ez = F * (D + 4) * scale * Q.abs() @ K.abs().t()
            t = torch.zeros_like(s)
            z = s
            if cap:
                t = torch.tanh(s / cap)
                z = cap * t
                ez = ez + 8 * F * cap
            if st['bias'] is not None:
                z = z + T[h][idx]
            live = z > -math.inf
            zf = torch.where(live, z, torch.zeros_like(z))
            ez = ez + 6 * F * zf.abs()
            p = torch.softmax(z, dim=-1)
            p = torch.where(live.any(1, keepdim=True), p,
                            torch.zeros_like(p))
            rp = 4 * ez.amax(1, keepdim=True) + (n + 16) * F
            rp = rp + 6 * F * zf.abs().amax(1, keepdim=True)
            o = p @ V
            pv = p @ V.abs()
            eo = (up + rp + n * F) * pv + u * o.abs()
            dp = G @ V.t()
            delta = (G * o).sum(1, keepdim=True)
            edp = (D + 2) * F * G.abs() @ V.abs().t()
            ed = (G.abs() * eo).sum(1, keepdim=True) + \
                D * F * (G * o).abs().sum(1, keepdim=True)
            dz = p * (dp - delta)
            edz = p * (rp * (dp - delta).abs() + edp + ed)
            ds = scale * (1 - t * t) * dz
            eds = scale * ((1 - t * t) * edz + dz.abs() * 16 * F) + \
                (up + 4 * F) * ds.abs()
            dq, dk, dv = ds @ K, ds.t() @ Q, p.t() @ G
            val['out'][sq, h], tol['out'][sq, h] = o, eo
            val['dq'][sq, h] = dq
            tol['dq'][sq, h] = eds @ K.abs() + n * F * ds.abs() @ K.abs()
            val['dk'][sk, g] += dk
            tol['dk'][sk, g] += eds.t() @ Q.abs() + \
                H * m * F * ds.t().abs() @ Q.abs()
            val['dv'][sk, g] += dv
            tol['dv'][sk, g] += ((up + rp + H * m * F) * p).t() @ G.abs()
            if st['bias'] is not None:
                val['dbias'][h].index_add_(0, idx.view(-1), dz.view(-1))
                tol['dbias'][h].index_add_(
                    0, idx.view(-1),
                    (edz + 64 * F * dz.abs()).view(-1))
    for n in ('dq', 'dk', 'dv'):
        tol[n] += u * val[n].abs()
    return val, tol


def _run(st, device, cap=0.0, scale=None, steps=1, grad=True, pack=False):
    dev = {n: (t.to(device) if t is not None else None)
           for n, t in st.items()}
    names = ['q', 'k', 'v'] + (['bias'] if dev['bias'] is not None else [])
    if grad:
        for n in names:
            dev[n].requires_grad_(True)
    same = st['ptr_k'] is st['ptr_q']
    out = segment_attention(
        dev['q'], dev['k'], dev['v'], dev['ptr_q'],
        None if same else dev['ptr_k'], scale=scale, cap=cap,
        bias=dev['bias'], pos_q=dev['pos_q'], pos_k=dev['pos_k'],
        octave_steps=steps)
    got = {'out': out.detach()}
    if grad:
        gs = torch.autograd.grad(out, [dev[n] for n in names], dev['do'])
        got.update(zip(['d' + n for n in names], gs))
    return {n: t.cpu() for n, t in got.items()}


def _close(got, val, tol, what=''):
    for n, t in got.items():
        assert torch.isfinite(t).all(), (what, n)
        err = (t.double() - val[n]).abs()
        # (1e-30: results below fp32's normal range)
        over = err - tol[n] - 1e-30
        worst = over.max().item() if over.numel() else 0.0
        assert worst <= 0, '{} {}: off by {:.3g}, allowed {:.3g}'.format(
            what, n, err.flatten()[over.argmax()],
            tol[n].flatten()[over.argmax()])


SHAPES = [
    # lq, lk (None: self), H, KV, D
    ([1], None, 1, 1, 32),
    ([1], [1], 1, 1, 8),
    ([3, 0, 19, 7], None, 4, 4, 64),
    ([5, 4, 0, 2], [3, 0, 6, 33], 2, 2, 32),
    ([31, 32, 33], [65, 64, 1], 2, 1, 64),
    ([40, 1, 130], None, 6, 2, 40),          # groups of 3: 30 rows a wave
    ([257], [300], 4, 1, 128),
    ([2, 1], [700, 1300], 8, 2, 128),        # few rows: split keys
    ([150], [140], 2, 2, 24),
    ([7, 9], None, 3, 1, 7),                 # unaligned rows
    ([129, 200], [66, 31], 1, 1, 128),
    ([129, 0, 200], [266, 40, 131], 2, 1, 64),   # long on both sides
    ([300], None, 3, 1, 20),
]


def _case(lq, lk, H, KV, D, dtype, **kw):
    st = _inputs(lq, lq if lk is None else lk, H, KV, D, dtype, **kw)
    if lk is None:
        st['ptr_k'] = st['ptr_q']
    return st


def test_bucket_starts_match_the_octave_count():
    for half, steps in ((3, 1), (15, 4), (7, 2), (31, 8), (0, 1), (22, 1)):
        starts = bucket_starts(half, steps)
        assert len(starts) == half + 1
        pos = torch.arange(-300, 300).int().view(-1, 1)
        zero = torch.zeros(1, 1, dtype=torch.int32)
        got = ref.position_buckets(zero, pos, starts).view(-1).tolist()
        want = [_plain_bucket(d, half, steps) for d in range(-300, 300)]
        assert got == want, (half, steps)


@pytest.mark.parametrize('lq,lk,H,KV,D', SHAPES)
def test_oracle_matches_plain_form(lq, lk, H, KV, D):
    if max(lq) > 200:
        lq = [min(x, 50) for x in lq]
    st = _case(lq, lk, H, KV, D, torch.float32, axes=1, half=3, tail=2)
    got = _run(st, 'cpu', cap=3.0)
    val, tol = _plain(st, cap=3.0, half=3)
    # (two fp32 forms: the kernel's bounds hold for torch's sums too)
    _close(got, val, tol)


def test_gradients_match_differences():
    st = _case([3, 2], [4, 0], 4, 2, 3, torch.float64, axes=2, half=1)
    st['bias'] = st['bias'].double()
    for n in ('q', 'k', 'v', 'bias'):
        st[n].requires_grad_(True)

    def f(q, k, v, bias):
        return segment_attention(q, k, v, st['ptr_q'], st['ptr_k'], cap=2.0,
                                 bias=bias, pos_q=st['pos_q'],
                                 pos_k=st['pos_k'])

    assert torch.autograd.gradcheck(f, (st['q'], st['k'], st['v'],
                                        st['bias']))


def test_rows_without_keys_are_zero():
    st = _case([2, 3], [0, 4], 1, 1, 4, torch.float32, tail=3)
    st['q'][:2] = float('nan')
    st['q'][5:] = float('inf')
    st['k'][4:] = float('nan')
    out = _run(st, 'cpu')
    assert (out['out'][:2] == 0).all() and (out['out'][5:] == 0).all()
    assert torch.isfinite(out['out']).all()
    assert (out['dq'][:2] == 0).all() and (out['dk'][4:] == 0).all()


def _bad_calls():
    q = torch.zeros(4, 2, 8)
    p = torch.tensor([0, 4], dtype=torch.int32)
    pos = torch.zeros(4, 1, dtype=torch.int32)
    t = torch.zeros(2, 3)
    return [
        dict(q=q[0], k=q, v=q, ptr_q=p),
        dict(q=q, k=q.double(), v=q, ptr_q=p),
        dict(q=q, k=q[:, :, :4], v=q[:, :, :4], ptr_q=p),
        dict(q=q, k=q, v=q[:3], ptr_q=p),
        dict(q=q[:, :1], k=q, v=q, ptr_q=p),
        dict(q=torch.zeros(4, 2, 200), k=torch.zeros(4, 2, 200),
             v=torch.zeros(4, 2, 200), ptr_q=p),
        dict(q=torch.zeros(4, 66, 8), k=torch.zeros(4, 2, 8),
             v=torch.zeros(4, 2, 8), ptr_q=p),
        dict(q=q, k=q, v=q, ptr_q=p.long()),
        dict(q=q, k=q, v=q, ptr_q=p, ptr_k=p[:1]),
        dict(q=q, k=q[:3], v=q[:3], ptr_q=p),
        dict(q=q, k=q, v=q, ptr_q=p, cap=-1.0),
        dict(q=q, k=q, v=q, ptr_q=p, cap=float('nan')),
        dict(q=q.int(), k=q.int(), v=q.int(), ptr_q=p),
        dict(q=q, k=q, v=q, ptr_q=p, bias=t),
        dict(q=q, k=q, v=q, ptr_q=p, bias=t, pos_q=pos.long()),
        dict(q=q, k=q, v=q, ptr_q=p, bias=t, pos_q=pos[:3]),
        dict(q=q, k=q, v=q, ptr_q=p, bias=t[:1], pos_q=pos),
        dict(q=q, k=q, v=q, ptr_q=p, bias=torch.zeros(2, 4), pos_q=pos),
        dict(q=q, k=q, v=q, ptr_q=p, bias=torch.zeros(2, 65), pos_q=pos),
        dict(q=q, k=q, v=q, ptr_q=p, bias=torch.zeros(2, 81),
             pos_q=pos.expand(4, 2)),
        dict(q=q, k=q, v=q, ptr_q=p, bias=torch.zeros(2, 27),
             pos_q=pos.expand(4, 3)),
        dict(q=q, k=q, v=q, ptr_q=p, bias=t, pos_q=pos, octave_steps=3),
        dict(q=q, k=q, v=q, ptr_q=p, bias=torch.zeros(2, 63), pos_q=pos,
             octave_steps=1),
    ]


@pytest.mark.parametrize('i', range(len(_bad_calls())))
def test_refusals(i):
    with pytest.raises(ValueError):
        segment_attention(**_bad_calls()[i])


# --------------------------------------------------------------------------
# GPU
# --------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('lq,lk,H,KV,D', SHAPES)
@pytest.mark.parametrize('cap,axes,half,steps', [
    (0.0, 0, 0, 1), (2.0, 1, 5, 2), (0.0, 2, 3, 1)])
def test_kernels_match_plain_form(lq, lk, H, KV, D, dtype, cap, axes, half,
                                  steps):
    st = _case(lq, lk, H, KV, D, dtype, axes=axes, half=half, tail=3)
    val, tol = _plain(st, cap=cap, half=half, steps=steps)
    _close(_run(st, 'cuda', cap=cap, steps=steps), val, tol, 'train')
    _close(_run(st, 'cuda', cap=cap, steps=steps, grad=False), val, tol,
           'forward')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_many_small_segments(dtype):
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 12, (700, ), generator=g).tolist()
    st = _case(lens, None, 2, 2, 32, dtype, axes=2, half=2)
    val, tol = _plain(st, half=2)
    _close(_run(st, 'cuda'), val, tol)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_strided_views_match_contiguous(dtype):
    g = torch.Generator().manual_seed(5)
    joint = torch.randn(50, 4 + 2 + 2, 32, generator=g).to(dtype).cuda()
    ptr = _ptr([20, 30]).cuda()
    q, k, v = joint[:, :4], joint[:, 4:6], joint[:, 6:]
    a = segment_attention(q, k, v, ptr)
    b = segment_attention(q.contiguous(), k.contiguous(), v.contiguous(),
                          ptr)
    assert torch.equal(a, b)
    # unaligned base, transposed heads, a last dimension that is not dense
    off = torch.zeros(50 * 4 * 32 + 1, dtype=dtype, device='cuda')
    off[1:] = q.reshape(-1)
    c = segment_attention(off[1:].view(50, 4, 32), k, v, ptr)
    assert torch.equal(a, c)
    d = segment_attention(q.permute(1, 2, 0).contiguous().permute(2, 0, 1),
                          k, v.transpose(0, 1).contiguous().transpose(0, 1),
                          ptr)
    assert torch.equal(a, d)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_padding_rows_and_empty_segments(dtype):
    """NaN and inf outside the segments never enter, rows without keys and
    behind the last segment are 0 - gradients too."""
    st = _case([2, 3, 40], [0, 4, 37], 2, 1, 32, dtype, tail=9, axes=1,
               half=2)
    val, tol = _plain(st, half=2)
    st['q'][45:], st['k'][41:], st['v'][41:] = (float('nan'), float('inf'),
                                                float('nan'))
    st['do'][45:] = float('nan')
    st['q'][:2] = float('nan')
    got = _run(st, 'cuda')
    for n in ('out', 'dq'):
        assert (got[n][:2] == 0).all() and (got[n][45:] == 0).all()
    for n in ('dk', 'dv'):
        assert (got[n][41:] == 0).all()
    _close(got, val, tol)


@pytest.mark.gpu
def test_masking_bias_values():
    """-inf entries mask their bucket (a row left with nothing gives 0), the
    type's lowest value masks unless it is everywhere (uniform then)."""
    st = _case([6, 40], None, 1, 1, 32, torch.float32, axes=1, half=2,
               span=4)
    st['bias'][:, [0, 4]] = -math.inf
    val, tol = _plain(st, half=2)
    _close(_run(st, 'cuda'), val, tol)
    st['bias'][:] = -math.inf
    got = _run(st, 'cuda')
    assert all((t == 0).all() for t in got.values())
    low = torch.finfo(torch.float32).min
    st['bias'][:] = 0.0
    st['bias'][:, [0, 4]] = low
    ninf = {n: t for n, t in st.items()}
    ninf['bias'] = st['bias'].clone()
    ninf['bias'][:, [0, 4]] = -math.inf
    a, b = _run(st, 'cuda', grad=False), _run(ninf, 'cuda', grad=False)
    alive = (_plain(ninf, half=2)[0]['out'] != 0).any(-1)
    assert torch.equal(a['out'][alive], b['out'][alive])
    st['bias'][:] = low
    out = _run(st, 'cuda', grad=False)['out']
    mean = torch.cat([s.mean(0, keepdim=True).expand_as(s)
                      for s in st['v'].split([6, 40])])
    assert torch.allclose(out, mean, rtol=0, atol=1e-6 * 4)


@pytest.mark.gpu
def test_far_positions():
    """Positions at int32's ends count as +-2^23; distances past fp32's
    integers stay in the last bucket."""
    st = _case([40], None, 1, 1, 32, torch.float32, axes=1, half=3)
    big = 2 ** 31 - 1
    st['pos_q'] = torch.tensor([[-big - 1], [big], [0], [1 << 23],
                                [-(1 << 23) + 1]] * 8, dtype=torch.int32)
    st['pos_k'] = st['pos_q'].flip(0).contiguous()
    val, tol = _plain(st, half=3)
    _close(_run(st, 'cuda'), val, tol)


@pytest.mark.gpu
def test_large_scores_do_not_overflow():
    for dtype in (torch.float32, torch.bfloat16):
        st = _case([70], None, 1, 1, 64, dtype, scale=30.0)
        out = _run(st, 'cuda')
        assert all(torch.isfinite(t).all() for t in out.values())
        # the largest score takes (nearly) all
        z = torch.einsum('ihd,jhd->ij', st['q'].double(), st['k'].double())
        best = st['v'][z.argmax(1), 0]
        gap = z.topk(2, dim=1)[0]
        clear = (gap[:, 0] - gap[:, 1]) / 8 > 40
        assert clear.any()
        # p v / l with one p: rounded p (bf16: 2^-8), the product, 1 / l,
        # its product and the output (bf16: 2^-8) - p itself cancels
        far = (out['out'][clear, 0].double() - best[clear].double()).abs()
        tol = 2 * _u(dtype) + 4 * F
        assert (far <= tol * best[clear].double().abs()).all()


@pytest.mark.gpu
def test_refusals_on_the_device():
    q = torch.zeros(4, 2, 8, device='cuda')
    p = torch.tensor([0, 4], dtype=torch.int32, device='cuda')
    with pytest.raises(ValueError):
        segment_attention(q.half(), q.half(), q.half(), p)
    with pytest.raises(ValueError):
        segment_attention(q, q, q, p.cpu())
    with pytest.raises(ValueError):
        segment_attention(q, q, q, p, bias=torch.zeros(2, 3, device='cuda'),
                          pos_q=torch.zeros(4, 1, dtype=torch.int32))


@pytest.mark.gpu
def test_empty_batches():
    p1 = torch.zeros(1, dtype=torch.int32, device='cuda')
    p2 = torch.zeros(3, dtype=torch.int32, device='cuda')
    for ptr in (p1, p2):
        q = torch.zeros(0, 2, 16, device='cuda', requires_grad=True)
        out = segment_attention(q, q, q, ptr)
        assert out.shape == (0, 2, 16)
        out.sum().backward()
        assert q.grad.shape == q.shape
    # queries without any key rows, and keys without any query
    q = torch.randn(5, 2, 16, device='cuda', requires_grad=True)
    k = torch.randn(0, 2, 16, device='cuda', requires_grad=True)
    ptr = torch.tensor([0, 5], dtype=torch.int32, device='cuda')
    z = torch.zeros(2, dtype=torch.int32, device='cuda')
    out = segment_attention(q, k, k, ptr, z)
    out.sum().backward()
    assert (out == 0).all() and (q.grad == 0).all()
    out = segment_attention(k, q, q, z, ptr)
    g, = torch.autograd.grad(out.sum(), q)
    assert out.shape == (0, 2, 16) and (g == 0).all()


@pytest.mark.gpu
def test_repeats_and_streams_are_bit_identical():
    st = _case([300, 20, 90], None, 4, 2, 64, torch.bfloat16, axes=1, half=7)
    a = _run(st, 'cuda', cap=5.0)
    b = _run(st, 'cuda', cap=5.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = _run(st, 'cuda', cap=5.0)
    torch.cuda.synchronize()
    for n in a:
        assert torch.equal(a[n], b[n]) and torch.equal(a[n], c[n]), n


@pytest.mark.gpu
def test_captured_step_follows_new_segments():
    """A captured forward + backward replays on new rows and NEW segments
    (ptr changed in place), eager work between the replays."""
    def make(lens, seed):
        st = _case(lens, None, 2, 2, 32, torch.float32, axes=1, half=3,
                   seed=seed, tail=60 - sum(lens))
        return st

    first = make([20, 30], 0)
    dev = {n: t.cuda() for n, t in first.items() if n != 'ptr_k'}
    leaves = [dev[n].requires_grad_(True) for n in ('q', 'k', 'v', 'bias')]

    def step():
        out = segment_attention(*leaves[:3], dev['ptr_q'], bias=leaves[3],
                                pos_q=dev['pos_q'], pos_k=dev['pos_k'])
        return [out.detach()] + list(
            torch.autograd.grad(out, leaves, dev['do']))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed, lens in enumerate(([20, 30], [1, 59], [50, 0], [33, 20])):
        new = make(lens, seed)
        with torch.no_grad():
            for n, t in dev.items():
                t.copy_(new[n])
        eager = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b), lens


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows whose offset passes 2^31 elements, 2^32 bytes (a strided view of
    a long cache)."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip('needs 16 GB')
    n, stride = 70, 1 << 26
    base = torch.zeros(n * stride // 2 + 64, dtype=torch.bfloat16,
                       device='cuda')
    k = base.as_strided((n, 1, 32), (stride // 2, 32, 1))
    g = torch.Generator().manual_seed(1)
    x = torch.randn(n, 1, 32, generator=g).to(torch.bfloat16).cuda()
    k.copy_(x)
    ptr = torch.tensor([0, n], dtype=torch.int32, device='cuda')
    assert torch.equal(segment_attention(x, k, k, ptr),
                       segment_attention(x, x, x, ptr))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('H,KV,D', [(1, 1, 128), (2, 1, 32), (3, 1, 64)])
def test_positions_in_order(dtype, H, KV, D):
    """Nodes in order, as a node ordering numbers them: whole blocks of
    pairs share a bucket, others cross from one to the next.  (400 keys: the
    sums of the table's gradient have 200 terms a lane and 256 columns, fewer
    than the n + 80 roundings its tolerance holds.)"""
    st = _case([400], None, H, KV, D, dtype, axes=1, half=7)
    for order in (torch.arange(400), torch.arange(400).flip(0) * 3 - 700):
        st['pos_q'] = st['pos_k'] = order.int().view(-1, 1)
        for steps in (1, 2):
            val, tol = _plain(st, cap=2.0, half=7, steps=steps)
            _close(_run(st, 'cuda', cap=2.0, steps=steps), val, tol)


@pytest.mark.gpu
def test_tiles_wider_than_a_buffers_range():
    """Row strides at which 64 rows of a tile stay within 2^31 bytes and 128
    do not."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip('needs 16 GB')
    n, stride = 200, 10 << 20
    base = torch.empty(n * stride, dtype=torch.bfloat16, device='cuda')
    wide = base.as_strided((n, 1, 32), (stride, 32, 1))
    g = torch.Generator().manual_seed(1)
    x = torch.randn(n, 1, 32, generator=g).to(torch.bfloat16).cuda()
    wide.copy_(x)
    ptr = torch.tensor([0, n], dtype=torch.int32, device='cuda')

    def run(t):
        leaf = t.detach().requires_grad_(True)
        out = segment_attention(leaf, leaf, leaf, ptr)
        return out, torch.autograd.grad(out, leaf, x)[0]

    for a, b in zip(run(wide), run(x)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('D', [5, 20, 66])
def test_padded_copies(dtype, D):
    """Rows that are no 16-byte chunks: few rows over long segments (split
    keys), long rows over few, and the step captured and replayed."""
    for lq, lk in (([2, 0, 1], [900, 7, 1400]), ([300], [40])):
        st = _case(lq, lk, 2, 1, D, dtype, axes=1, half=3, tail=2)
        val, tol = _plain(st, cap=3.0, half=3)
        _close(_run(st, 'cuda', cap=3.0), val, tol)
    dev = {n: t.cuda() for n, t in st.items()}
    leaves = [dev[n].requires_grad_(True) for n in ('q', 'k', 'v')]

    def step():
        out = segment_attention(*leaves, dev['ptr_q'], dev['ptr_k'])
        return [out.detach()] + list(
            torch.autograd.grad(out, leaves, dev['do']))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        with torch.no_grad():
            for t in leaves:
                t.mul_(0.9).add_(0.1 * seed)
        eager = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_captured_graphs_and_eager_calls_share_nothing():
    """Two captured calls with split keys and one eager call, replayed in
    turn: no workspace of one is another's."""
    st = [_case([2, 1], [3000, 2500], 4, 1, 64, torch.bfloat16, seed=s)
          for s in range(3)]
    dev = [{n: t.cuda() for n, t in d.items() if t is not None} for d in st]

    def call(d):
        return segment_attention(d['q'], d['k'], d['v'], d['ptr_q'],
                                 d['ptr_k'])

    want = [call(d).clone() for d in dev]
    graphs, outs = [], []
    for d in dev[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(d))
        graphs.append(g)
    for _ in range(3):
        graphs[1].replay()
        graphs[0].replay()
        e = call(dev[2])
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0])
        assert torch.equal(outs[1], want[1])
        assert torch.equal(e, want[2])


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    q = torch.randn(5, 1, 16, device='cuda', requires_grad=True)
    ptr = torch.tensor([0, 5], dtype=torch.int32, device='cuda')
    g, = torch.autograd.grad(segment_attention(q, q, q, ptr).sum(), q,
                             create_graph=True)
    with pytest.raises(RuntimeError, match='differentiated again'):
        g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('axes,cap', [(0, 0.0), (1, 2.0)])
@pytest.mark.parametrize('what', ['q', 'k', 'v', 'do'])
def test_non_finite_segments_stay_alone(dtype, axes, cap, what):
    """NaN and inf in some segments' rows never reach the segments that
    share tiles with them (rows and keys of a tile are consecutive rows,
    whatever their segments)."""
    lens = [5, 7, 0, 40, 3, 60, 1, 1, 150]
    st = _case(lens, [9, 4, 3, 30, 0, 80, 2, 1, 90], 2, 1, 32, dtype,
               axes=axes, half=2, tail=4)
    val, tol = _plain(st, cap=cap, half=2)
    pq, pk = st['ptr_q'].tolist(), st['ptr_k'].tolist()
    own = pq if what in ('q', 'do') else pk
    st[what][own[1] + 1] = float('nan')
    st[what][own[5]:own[5] + 40] = math.inf
    got = _run(st, 'cuda', cap=cap)
    for n, t in got.items():
        if n == 'dbias':        # the bad rows' own contribution
            continue
        ptr = pq if n in ('out', 'dq') else pk
        for b in range(len(lens)):
            rows = slice(ptr[b], ptr[b + 1])
            if b in (1, 5):
                continue
            err = (t[rows].double() - val[n][rows]).abs()
            assert (err <= tol[n][rows] + 1e-30).all(), (n, b)
    bad = {'q': ('out', 'dq', 'dk'), 'k': ('out', 'dq', 'dk'),
           'v': ('out', 'dq', 'dk'), 'do': ('dq', 'dk', 'dv')}[what]
    for n in bad:
        ptr = pq if n in ('out', 'dq') else pk
        assert not torch.isfinite(got[n][ptr[1]:ptr[2]]).all(), n


@pytest.mark.gpu
def test_many_empty_segments_between_rows():
    """More boundaries than lanes between two rows of a tile."""
    lens = [3] + [0] * 200 + [2] + [0] * 70 + [5, 0, 0, 1] + [0] * 64 + [4]
    st = _case(lens, None, 2, 2, 32, torch.float32)
    val, tol = _plain(st)
    _close(_run(st, 'cuda'), val, tol)
