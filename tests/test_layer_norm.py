"""Layer norm (ops/norm.py, csrc/hip/layer_norm.hip) against a plain form in
64 bits.  Tolerances carry the arithmetic: fp32 sums of C (or of the rows)
terms, at most as many 2^-24 steps as terms, and one rounding of each output
to its type."""
import pytest
import torch

from deep_graph_matching_consensus_amd.ops import layer_norm

F = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _case(shape, dtype, residual, seed=0, shift=0.3, scale=1.5):
    g = torch.Generator().manual_seed(seed)

    def rnd(*s, k=1.0, c=0.0, dt=dtype):
        return (torch.randn(s, generator=g) * k + c).to(dt)

    C = shape[-1]
    st = dict(x=rnd(*shape, k=scale, c=shift), w=rnd(C, k=0.3, c=1.0,
                                                     dt=torch.float32),
              b=rnd(C, k=0.3, dt=torch.float32), dy=rnd(*shape), res=None,
              ds=None)
    if residual:
        st['res'], st['ds'] = rnd(*shape), rnd(*shape)
    return st


def _plain(st, eps=1e-5):
    """Values and error bounds."""
    dt = st['x'].dtype
    u = torch.finfo(dt).eps / 2
    C = st['x'].size(-1)
    s = st['x'].double().reshape(-1, C)
    val, tol = {}, {}
    if st['res'] is not None:
        # the sum's own rounding: the oracle rounds the same fp32 sum
        s = (st['x'].float() + st['res'].float()).to(dt)
        val['s'] = s.reshape(-1, C).double()
        tol['s'] = torch.zeros_like(val['s'])
        s = val['s']
    w, b = st['w'].double(), st['b'].double()
    R = s.size(0)
    mean = s.mean(1, keepdim=True)
    var = ((s - mean) ** 2).mean(1, keepdim=True)
    std = (var + eps).sqrt()
    n = (s - mean) / std
    # mean: C steps; (x - mean)^2 and its sum; rsqrt, products
    em = (C + 1) * F * s.abs().mean(1, keepdim=True)
    rel = (C + 12) * F + em / std + em ** 2 / (var + eps)
    en = (em + 2 * F * (s - mean).abs()) / std + rel * n.abs()
    y = n * w + b
    val['y'] = y
    tol['y'] = en * w.abs() + 4 * F * (y.abs() + b.abs()) + u * y.abs()
    dy = st['dy'].double().reshape(-1, C)
    h = dy * w
    c1, c2 = h.mean(1, keepdim=True), (h * n).mean(1, keepdim=True)
    dx = (h - c1 - n * c2) / std
    e1 = (C + 2) * F * h.abs().mean(1, keepdim=True)
    e2 = (C + 3) * F * (h * n).abs().mean(1, keepdim=True) + \
        (h.abs() * en).mean(1, keepdim=True)
    edx = (e1 + en * c2.abs() + n.abs() * e2 +
           4 * F * (h.abs() + c1.abs() + (n * c2).abs())) / std + \
        rel * dx.abs()
    if st['res'] is not None:
        dx = dx + st['ds'].double().reshape(-1, C)
        edx = edx + 2 * F * dx.abs()
        val['dres'], tol['dres'] = dx, edx + u * dx.abs()
    val['dx'], tol['dx'] = dx, edx + u * dx.abs()
    val['dw'], val['db'] = (dy * n).sum(0), dy.sum(0)
    tol['dw'] = (R + 2) * F * (dy * n).abs().sum(0) + (dy.abs() * en).sum(0)
    tol['db'] = (R + 1) * F * dy.abs().sum(0)
    return val, tol


def _run(st, device, grad=True):
    dev = {n: None if t is None else t.to(device) for n, t in st.items()}
    names = ['x', 'w', 'b'] + (['res'] if st['res'] is not None else [])
    if grad:
        for n in names:
            dev[n].requires_grad_(True)
    out = layer_norm(dev['x'], dev['w'], dev['b'], residual=dev['res'])
    out = dict(zip(('y', 's'), out if st['res'] is not None else (out, )))
    got = {n: t.detach() for n, t in out.items()}
    if grad:
        outs = [out['y']] + ([out['s']] if 's' in out else [])
        gs = [dev['dy']] + ([dev['ds']] if 's' in out else [])
        got.update(zip(['d' + n for n in names], torch.autograd.grad(
            outs, [dev[n] for n in names], gs)))
    C = st['x'].size(-1)
    return {n: t.cpu().reshape(-1, C) if t.dim() > 1 else t.cpu()
            for n, t in got.items()}


def _close(got, val, tol):
    for n, t in got.items():
        err = (t.double() - val[n]).abs()
        # (fp16 outputs below its normal range: half a subnormal step)
        low = 2.0 ** -25 if t.dtype == torch.float16 else 1e-30
        over = err - tol[n] - low
        assert over.numel() == 0 or over.max() <= 0, (
            n, err.flatten()[over.argmax()], tol[n].flatten()[over.argmax()])


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 16), (33, 64), (2, 3, 65), (20, 256),
          (7, 300), (9, 511), (4, 512), (6, 1024), (5, 1025), (3, 2048),
          (3, 2050), (2, 4096), (2, 8192), (2, 8191), (0, 32), (1500, 40),
          (3000, 128)]


@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('shape', SHAPES[:10])
def test_oracle_matches_plain_form(shape, residual):
    st = _case(shape, torch.float32, residual)
    _close(_run(st, 'cpu'), *_plain(st))


def test_gradients_match_differences():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(4, 6, generator=g, dtype=torch.float64)
    r = torch.randn(4, 6, generator=g, dtype=torch.float64)
    w = torch.randn(6, generator=g, dtype=torch.float64)
    b = torch.randn(6, generator=g, dtype=torch.float64)
    args = [t.requires_grad_(True) for t in (x, w, b, r)]
    assert torch.autograd.gradcheck(
        lambda x, w, b, r: layer_norm(x, w, b, residual=r), args)


@pytest.mark.parametrize('kw', [
    dict(x=torch.zeros(3, 0)), dict(x=torch.zeros(2, 8193)),
    dict(x=torch.zeros(3, 4, dtype=torch.int32)),
    dict(x=torch.zeros(3, 4), weight=torch.ones(3)),
    dict(x=torch.zeros(3, 4), bias=torch.ones(4)),
    dict(x=torch.zeros(3, 4), weight=torch.ones(4), bias=torch.ones(5)),
    dict(x=torch.zeros(3, 4), weight=torch.ones(4).int()),
    dict(x=torch.zeros(3, 4), eps=0.0),
    dict(x=torch.zeros(3, 4), residual=torch.zeros(4)),
    dict(x=torch.zeros(3, 4), residual=torch.zeros(3, 4).half()),
    dict(x=torch.zeros(()))])
def test_refusals(kw):
    with pytest.raises(ValueError):
        layer_norm(**kw)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('shape', SHAPES)
def test_kernels_match_plain_form(shape, residual, dtype):
    st = _case(shape, dtype, residual)
    val, tol = _plain(st)
    _close(_run(st, 'cuda'), val, tol)
    _close(_run(st, 'cuda', grad=False), val, tol)


@pytest.mark.gpu
def test_constant_rows_and_large_offsets():
    """A constant row gives its bias; a large common offset keeps the
    variance's precision (two passes)."""
    x = torch.full((4, 96), 3.0, device='cuda')
    w, b = torch.ones(96, device='cuda'), torch.arange(96., device='cuda')
    assert torch.equal(layer_norm(x, w, b), b.expand(4, 96))
    st = _case((6, 256), torch.float32, False, shift=1000.0, scale=1.0)
    _close(_run(st, 'cuda'), *_plain(st))


@pytest.mark.gpu
def test_strides_views_and_parameter_types():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(50, 96, generator=g).cuda()
    want = layer_norm(x[:, :64].contiguous())
    assert torch.equal(layer_norm(x[:, :64]), want)
    flat = torch.zeros(50 * 64 + 1, device='cuda')
    flat[1:] = x[:, :64].reshape(-1)
    off = layer_norm(flat[1:].view(50, 64))         # unaligned rows
    assert (off - want).abs().max() <= 64 * F * 8
    w = torch.randn(64, generator=g).cuda()
    a = layer_norm(x[:, :64], w.bfloat16().requires_grad_(True))
    assert torch.equal(a, layer_norm(x[:, :64], w.bfloat16().float()))
    wb = w.bfloat16().requires_grad_(True)
    gw, = torch.autograd.grad(layer_norm(x[:, :64], wb).sum(), wb)
    assert gw.dtype == torch.bfloat16


@pytest.mark.gpu
def test_partial_gradients():
    """Only some inputs want gradients, only some outputs give one."""
    st = _case((40, 48), torch.float32, True)
    val, tol = _plain(st)
    dev = {n: t.cuda() for n, t in st.items()}
    x = dev['x'].clone().requires_grad_(True)
    y, s = layer_norm(x, dev['w'], dev['b'], residual=dev['res'])
    gx, = torch.autograd.grad([y, s], x, [dev['dy'], dev['ds']])
    _close({'dx': gx.cpu()}, val, tol)
    y, s = layer_norm(x, dev['w'], dev['b'], residual=dev['res'])
    gx, = torch.autograd.grad(s, x, dev['ds'])
    assert torch.equal(gx, dev['ds'])
    w = dev['w'].clone().requires_grad_(True)
    y = layer_norm(dev['x'], w)
    gw, = torch.autograd.grad(y, w, dev['dy'])
    plain = dict(st, res=None, ds=None)
    val, tol = _plain(plain)
    _close({'dw': gw.cpu()}, val, tol)


@pytest.mark.gpu
def test_repeats_and_captured_replays_are_identical():
    st = _case((3000, 256), torch.bfloat16, True)
    dev = {n: t.cuda() for n, t in st.items()}
    leaves = [dev[n].requires_grad_(True) for n in ('x', 'res', 'w', 'b')]

    def step():
        y, s = layer_norm(dev['x'], dev['w'], dev['b'], residual=dev['res'])
        return [y.detach(), s.detach()] + list(torch.autograd.grad(
            [y, s], leaves, [dev['dy'], dev['ds']]))

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
        new = _case((3000, 256), torch.bfloat16, True, seed=seed)
        with torch.no_grad():
            for n, t in dev.items():
                t.copy_(new[n])
        eager = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x = torch.randn(3, 16, device='cuda', requires_grad=True)
    g, = torch.autograd.grad(layer_norm(x).square().sum(), x,
                             create_graph=True)
    with pytest.raises(RuntimeError, match='differentiated again'):
        g.sum().backward()
