"""The attentional operators together: layers of ``nn.AttentionConv`` (norm,
attention, position bias) over packed pairs, the pairs' scores, and the
matches' log-probabilities as a loss - against a dense form in 64 bits graph
by graph - and ``DGMC.log_probs``.

Tolerances of the chain: each of the two layers and the score product carries
fp32 rounding (2^-24 a step) through sums of at most ``S`` = 64 terms and
products of 32 channels; with inputs of order one every intermediate stays
below 16, so 16 * S * 2^-24 per stage over 8 stages bounds values, and the
same relative to the largest gradient entry bounds gradients.
"""
import math

import pytest
import torch

from deep_graph_matching_consensus_amd.models import DGMC, GIN
from deep_graph_matching_consensus_amd.nn import AttentionConv
from deep_graph_matching_consensus_amd.ops import match_log_probs
from deep_graph_matching_consensus_amd.ops import reference as ref
from deep_graph_matching_consensus_amd.ops.attention import bucket_starts

TOL = 8 * 16 * 64 * 2.0 ** -24
N_S, N_T = [7, 1, 12, 5], [9, 4, 12, 1]


def _batch(lens):
    return torch.repeat_interleave(torch.arange(len(lens)),
                                   torch.tensor(lens))


def _setup(seed=0):
    g = torch.Generator().manual_seed(seed)
    torch.manual_seed(seed)
    convs = torch.nn.ModuleList([
        AttentionConv(32, 4, key_heads=2, cap=4.0, axes=2, half=2),
        AttentionConv(32, 4, key_heads=2, cap=4.0, axes=2, half=2)])
    for c in convs:
        c.table.data.normal_(generator=g)
        c.norm_bias.data.normal_(0, 0.1, generator=g)
    x = [torch.randn(sum(n), 32, generator=g) for n in (N_S, N_T)]
    pos = [torch.randint(0, 9, (sum(n), 2), generator=g, dtype=torch.int32)
           for n in (N_S, N_T)]
    y = torch.cat([torch.randint(0, t, (s, ), generator=g)
                   for s, t in zip(N_S, N_T)])
    return convs, x, pos, y


def _loss(r):
    return -r.log_prob.mean() + 0.1 * r.entropy.mean()


def _packed(convs, x, pos, y):
    """As a user calls it: self-attention, then cross-attention."""
    dev = x[0].device
    b_s, b_t = _batch(N_S).to(dev), _batch(N_T).to(dev)
    h_s = convs[0](x[0], b_s, pos[0])
    h_t = convs[0](x[1], b_t, pos[1])
    o_s = convs[1](h_s, b_s, pos[0], other=(h_t, b_t, pos[1]))
    rows = []
    s = t = 0
    for n, m in zip(N_S, N_T):
        z = o_s[s:s + n] @ h_t[t:t + m].t() / 32
        rows.append(torch.nn.functional.pad(z, (0, max(N_T) - m)))
        s, t = s + n, t + m
    n_cols = torch.tensor(N_T, dtype=torch.int32)[_batch(N_S)].to(dev)
    return match_log_probs(torch.cat(rows), y, n_cols, top=1)


def _attend(conv, x, x_o, pos, pos_o):
    """One graph, 64 bits, straight from the formulas."""
    def norm(v):
        d = v - v.mean(-1, keepdim=True)
        return d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * \
            conv.norm_weight.double() + conv.norm_bias.double()

    def lin(v, m):
        return v @ m.weight.double().t() + m.bias.double()

    q = lin(norm(x), conv.query).view(-1, 4, 8)
    kv = lin(norm(x_o), conv.key_value).view(-1, 4, 8)
    idx = ref.position_buckets(pos, pos_o, bucket_starts(2))
    outs = []
    for h in range(4):
        z = q[:, h] @ kv[:, h // 2].t() / math.sqrt(8)
        z = 4.0 * torch.tanh(z / 4.0) + conv.table.double()[h][idx]
        outs.append(torch.softmax(z, -1) @ kv[:, 2 + h // 2])
    return x + lin(torch.cat(outs, -1), conv.out)


def _plain(convs, x, pos, y):
    s = t = 0
    logp, ent, best = [], [], []
    for n, m in zip(N_S, N_T):
        xs, xt = x[0][s:s + n].double(), x[1][t:t + m].double()
        ps, pt = pos[0][s:s + n], pos[1][t:t + m]
        hs = _attend(convs[0], xs, xs, ps, ps)
        ht = _attend(convs[0], xt, xt, pt, pt)
        lp = torch.log_softmax(
            _attend(convs[1], hs, ht, ps, pt) @ ht.t() / 32, -1)
        logp.append(lp.gather(1, y[s:s + n].view(-1, 1)).view(-1))
        ent.append(-(lp.exp() * lp).sum(-1))
        best.append(lp.argmax(-1))
        s, t = s + n, t + m
    return torch.cat(logp), torch.cat(ent), torch.cat(best)


def _compare(device):
    convs, x, pos, y = _setup()
    logp, ent, best = _plain(convs, x, pos, y)
    params = list(convs.parameters())
    want = torch.autograd.grad(-logp.mean() + 0.1 * ent.mean(), params)
    convs = convs.to(device)
    r = _packed(convs, [t.to(device) for t in x],
                [p.to(device) for p in pos], y.to(device))
    assert torch.equal(r.top_index.view(-1).cpu(), best)
    assert (r.log_prob.cpu().double() - logp).abs().max() < TOL
    assert (r.entropy.cpu().double() - ent).abs().max() < TOL
    got = torch.autograd.grad(_loss(r), list(convs.parameters()))
    for g, w in zip(got, want):
        assert (g.cpu().double() - w).abs().max() <= \
            TOL * max(1e-2, w.abs().max())


def test_layers_and_loss_match_a_dense_form():
    _compare('cpu')


@pytest.mark.gpu
def test_layers_and_loss_match_a_dense_form_on_the_gpu():
    _compare('cuda')


@pytest.mark.gpu
def test_layers_under_autocast():
    """bf16 projections and attention: finite, near the fp32 result (two
    layers of bf16 rounding, 2^-8 each step of order one)."""
    convs, x, pos, y = _setup(1)
    convs = convs.cuda()
    args = ([t.cuda() for t in x], [p.cuda() for p in pos], y.cuda())
    want = _packed(convs, *args)
    with torch.autocast('cuda', torch.bfloat16):
        got = _packed(convs, *args)
    assert torch.isfinite(got.log_prob).all()
    assert (got.log_prob - want.log_prob).abs().max() < 32 * 2.0 ** -8
    grads = torch.autograd.grad(_loss(got), list(convs.parameters()))
    assert all(torch.isfinite(g).all() for g in grads)


def test_layer_repr_and_reset():
    conv = AttentionConv(32, 4, key_heads=2, cap=4.0, axes=1)
    assert repr(conv) == ('AttentionConv(32, heads=4, key_heads=2, cap=4.0, '
                          'axes=1)')
    conv.table.data.fill_(3.0)
    conv.reset_parameters()
    assert (conv.table == 0).all() and conv.table.shape == (4, 7)


# --------------------------------------------------------------------------
# DGMC.log_probs
# --------------------------------------------------------------------------
def _graphs(device, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens_s, lens_t = [6, 4, 9], [8, 4, 10]

    def side(lens):
        x = torch.randn(sum(lens), 16, generator=g)
        ei, a = [], 0
        for n in lens:
            ei.append(torch.randint(0, n, (2, 3 * n), generator=g) + a)
            a += n
        return (x.to(device), torch.cat(ei, 1).to(device), None,
                _batch(lens).to(device))

    s, t = side(lens_s), side(lens_t)
    y = torch.cat([torch.randint(0, n, (m, ), generator=g)
                   for m, n in zip(lens_s, lens_t)]).to(device)
    y[3] = -1
    return s + t, y


def _check_dgmc(device, k):
    torch.manual_seed(0)
    model = DGMC(GIN(16, 16, 2), GIN(8, 8, 2), num_steps=2, k=k).to(device)
    model.eval()
    args, y = _graphs(device)
    torch.manual_seed(1)
    with torch.no_grad():
        S = model(*args)
    torch.manual_seed(1)
    with torch.no_grad():
        res = model.log_probs(*args, y_col=y, top=3)
    rows = torch.arange(y.numel(), device=device)
    for s, r in zip(S, res):
        p = s.to_dense() if s.is_sparse else s
        want = p[rows, y.clamp(min=0)].double().log()
        want[y < 0] = 0.0
        fin = torch.isfinite(want)
        assert torch.equal(fin, torch.isfinite(r.log_prob))
        # (the probabilities are rounded: 2^-24 and the softmax's own sums)
        assert (r.log_prob.double() - want)[fin].abs().max() < 64 * 2 ** -24 \
            * 16
        q = p.double()
        ent = -(q * torch.where(q > 0, q, torch.ones_like(q)).log()).sum(-1)
        assert (r.entropy.double() - ent).abs().max() < 1e-5
        val, idx = p.sort(dim=-1, descending=True, stable=True)
        assert torch.equal(r.top_index[:, 0], idx[:, 0])
        assert (r.top_log_prob.double().exp() - val[:, :3].double()
                ).abs().max() < 64 * 2 ** -24


@pytest.mark.parametrize('k', [-1, 3])
def test_dgmc_log_probs_match_forward(k):
    _check_dgmc('cpu', k)


@pytest.mark.gpu
@pytest.mark.parametrize('k', [-1, 3])
def test_dgmc_log_probs_match_forward_on_the_gpu(k):
    _check_dgmc('cuda', k)


@pytest.mark.gpu
@pytest.mark.parametrize('k', [-1, 3])
def test_dgmc_log_probs_under_autocast(k):
    """The scores of the model's own bf16 path: the same as its
    probabilities'."""
    torch.manual_seed(0)
    model = DGMC(GIN(16, 16, 2), GIN(8, 8, 2), num_steps=2, k=k).cuda().eval()
    args, y = _graphs('cuda')
    with torch.no_grad(), torch.autocast('cuda', torch.bfloat16):
        torch.manual_seed(1)
        S = model(*args)
        torch.manual_seed(1)
        res = model.log_probs(*args, y_col=y, top=2)
    for s, r in zip(S, res):
        p = s.to_dense() if s.is_sparse else s
        best = p.max(dim=-1).values.double()
        # (both softmaxes are fp32 on the same scores)
        assert (r.top_log_prob[:, 0].double().exp() - best).abs().max() < \
            64 * 2 ** -24


def test_dgmc_log_probs_train_and_refuse_sinkhorn():
    args, y = _graphs('cpu')
    model = DGMC(GIN(16, 16, 2), GIN(8, 8, 2), num_steps=1)
    first, last = model.log_probs(*args, y_col=y)
    grads = torch.autograd.grad(-(first.log_prob + last.log_prob).mean(),
                                list(model.psi_1.parameters()),
                                allow_unused=True)
    assert all(torch.isfinite(g).all() for g in grads if g is not None)
    model = DGMC(GIN(16, 16, 2), GIN(8, 8, 2), num_steps=1,
                 normalization='sinkhorn')
    with pytest.raises(ValueError):
        model.log_probs(*args)
