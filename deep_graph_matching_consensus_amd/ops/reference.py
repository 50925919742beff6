"""Pure-PyTorch oracles for every native op (CPU path + test reference).

These follow the reference semantics literally (same math, same op order as
``/root/reference/dgmc/models/dgmc.py`` and the PyG/torch_scatter/
torch_spline_conv call sites it relies on).  The HIP kernels in ``csrc/hip``
are validated against these in fp32.
"""
import torch


# --------------------------------------------------------------------------
# Message passing
# --------------------------------------------------------------------------
def sum_dtype(dtype):
    """The type in which values of ``dtype`` are summed: fp64 ones in fp64
    (a fp64 model's oracle keeps all its bits), all others in fp32."""
    return dtype if dtype == torch.float64 else torch.float32


def spmm(row, col, val, num_rows, x, self_x=None, self_scale=None,
         bias=None, relu=False, out_dtype=torch.float32):
    # 64-bit inputs (a 64-bit oracle) sum in 64 bits: index_add_ adds in any
    # order on the GPU, and in 32 bits that order decides the sign of a value
    # of 1e-7 - a ReLU, and with it a gradient, differently from run to run.
    acc = sum_dtype(x.dtype)
    xf = x.to(acc)
    out = torch.zeros(num_rows, x.size(1), dtype=acc, device=x.device)
    if col.numel() > 0:
        out.index_add_(0, row.long(), val.to(acc).view(-1, 1) *
                       xf[col.long()])
    if self_x is not None:
        out = out + self_scale.to(acc) * self_x.to(acc)
    if bias is not None:
        out = out + bias.to(acc)
    if relu:
        out = torch.relu(out)
    return out.to(out_dtype)


def spline_basis(pseudo, kernel_size, is_open_spline, degree=1):
    r"""Open/closed B-spline basis (torch_spline_conv ``spline_basis``).

    Returns ``basis [E, S]`` (fp32) and ``weight_index [E, S]`` (int64) with
    ``S = (degree + 1) ** dim``.
    """
    pseudo = pseudo.view(-1, 1) if pseudo.dim() == 1 else pseudo
    E, dim = pseudo.shape
    S = (degree + 1) ** dim
    device = pseudo.device
    s = torch.arange(S, device=device)
    basis = torch.ones(E, S, dtype=torch.float32, device=device)
    wi = torch.zeros(E, S, dtype=torch.long, device=device)
    offset = 1
    for d in range(dim):
        k_mod = (s // ((degree + 1) ** d)) % (degree + 1)          # [S]
        ks = int(kernel_size[d])
        v = pseudo[:, d].float() * (ks - degree * int(is_open_spline[d]))
        fl = v.floor()
        wi = wi + ((fl.long().view(-1, 1) + k_mod.view(1, -1)) % ks) * offset
        offset *= ks
        v = (v - fl).view(-1, 1)
        basis = basis * _basis_fn(v, k_mod.view(1, -1), degree)
    return basis, wi


def _basis_fn(v, k_mod, degree):
    if degree == 1:
        return 1 - v - k_mod + 2 * v * k_mod
    if degree == 2:
        b0 = 0.5 * v * v - v + 0.5
        b1 = -v * v + v + 0.5
        b2 = 0.5 * v * v
        return torch.where(k_mod == 0, b0, torch.where(k_mod == 1, b1, b2))
    if degree == 3:
        b0 = (1 - v) ** 3 / 6.
        b1 = (3 * v ** 3 - 6 * v ** 2 + 4) / 6.
        b2 = (-3 * v ** 3 + 3 * v ** 2 + 3 * v + 1) / 6.
        b3 = v ** 3 / 6.
        return torch.where(k_mod == 0, b0, torch.where(
            k_mod == 1, b1, torch.where(k_mod == 2, b2, b3)))
    raise ValueError('degree must be 1, 2 or 3')


# --------------------------------------------------------------------------
# Dense correspondence (dgmc.py:15-19, 161-183)
# --------------------------------------------------------------------------
def masked_softmax(src, mask, dim=-1):
    out = src.masked_fill(~mask, float('-inf'))
    out = torch.softmax(out, dim=dim)
    out = out.masked_fill(~mask, 0)
    return out


def masked_sinkhorn(src, mask, num_iters=10, tau=1.0):
    r"""Log-domain Sinkhorn normalisation over the valid entries (opt-in
    extension; the reference only uses row softmax).

    Alternates row and column normalisation of ``exp(src / tau)`` and ends
    with a row normalisation, so every valid row sums to 1 like
    :func:`masked_softmax` while columns are pushed towards 1.  Invalid
    entries are 0; fully masked rows/columns stay 0 (no NaN).
    """
    neg = torch.finfo(src.dtype).min / 4
    log = (src / tau).masked_fill(~mask, neg)
    for _ in range(num_iters):
        log = log - torch.logsumexp(log, dim=-1, keepdim=True)
        log = log.masked_fill(~mask, neg)
        log = log - torch.logsumexp(log, dim=-2, keepdim=True)
        log = log.masked_fill(~mask, neg)
    log = log - torch.logsumexp(log, dim=-1, keepdim=True)
    return log.exp().masked_fill(~mask, 0)


def count_mask(n_s, n_t, N_s, N_t):
    """``[B, N_s, N_t]`` validity mask from per-pair node counts."""
    device = n_s.device
    ms = torch.arange(N_s, device=device).view(1, -1) < n_s.view(-1, 1).long()
    mt = torch.arange(N_t, device=device).view(1, -1) < n_t.view(-1, 1).long()
    return ms.view(-1, N_s, 1) & mt.view(-1, 1, N_t)


def consensus_mlp_dense(o_s, o_t, W1, b1, W2, b2):
    """``MLP(o_s[:, :, None] - o_t[:, None])`` exactly as dgmc.py:178-179."""
    B, N_s, R = o_s.shape
    N_t = o_t.size(1)
    D = o_s.view(B, N_s, 1, R) - o_t.view(B, 1, N_t, R)
    h = torch.relu(torch.nn.functional.linear(D, W1, b1))
    return torch.nn.functional.linear(h, W2, b2).squeeze(-1)


def consensus_mlp_sparse(o_s, o_t_gathered, W1, b1, W2, b2):
    """``MLP(o_s[:, :, None] - o_t[S_idx])`` as dgmc.py:219-223."""
    D = o_s.unsqueeze(2) - o_t_gathered
    h = torch.relu(torch.nn.functional.linear(D, W1, b1))
    return torch.nn.functional.linear(h, W2, b2).squeeze(-1)


def top_k(x_s, x_t, k):
    """Indices of the k largest inner products, best first (dgmc.py:85-94)."""
    S_ij = x_s @ x_t.transpose(-1, -2)
    return S_ij.topk(k, dim=2)[1]


# --------------------------------------------------------------------------
# Attention inside the segments of a packed batch
# --------------------------------------------------------------------------
def position_buckets(pos_q, pos_k, starts):
    """``[n_q, n_k]`` column of the bias table of every pair of positions
    (``[n, axes]``): ``half +- b`` per axis, the first axis most significant;
    ``b`` is the last bucket of ``starts`` not beyond the distance."""
    half = len(starts) - 1
    edges = torch.tensor(starts[1:], dtype=torch.long, device=pos_q.device)
    lim = 1 << 23
    out = torch.zeros((pos_q.size(0), pos_k.size(0)), dtype=torch.long,
                      device=pos_q.device)
    for x in range(pos_q.size(1)):
        d = pos_k[:, x].long().clamp(-lim, lim).view(1, -1) - \
            pos_q[:, x].long().clamp(-lim, lim).view(-1, 1)
        b = (d.abs().unsqueeze(-1) >= edges).sum(-1)
        out = out * (2 * half + 1) + half + torch.sign(d) * b
    return out


def segment_attention(q, k, v, ptr_q, ptr_k, scale, cap=0.0, bias=None,
                      pos_q=None, pos_k=None, starts=(0, )):
    """Attention of every segment's rows over its keys, in fp32 (fp64 for
    fp64 inputs), rounded once to ``q``'s dtype."""
    acc = torch.float64 if q.dtype == torch.float64 else torch.float32
    G = q.size(1) // k.size(1)
    qa, ka, va = q.to(acc), k.to(acc), v.to(acc)
    pq, pk = ptr_q.tolist(), ptr_k.tolist()
    outs, rows = [], 0
    never = torch.ones((), dtype=torch.bool, device=q.device)
    for b in range(len(pq) - 1):
        sq, sk = slice(pq[b], pq[b + 1]), slice(pk[b], pk[b + 1])
        rows = pq[b + 1]
        if pq[b + 1] == pq[b]:
            continue
        if pk[b + 1] == pk[b]:
            outs.append(qa[sq].masked_fill(never, 0))
            continue
        qs = qa[sq].transpose(0, 1)
        ks = ka[sk].repeat_interleave(G, dim=1).transpose(0, 1)
        vs = va[sk].repeat_interleave(G, dim=1).transpose(0, 1)
        z = scale * (qs @ ks.transpose(1, 2))
        if cap:
            z = cap * torch.tanh(z / cap)
        if bias is not None:
            z = z + bias.to(acc).clamp(min=-1e38).where(
                bias > -float('inf'), bias.to(acc))[
                    :, position_buckets(pos_q[sq], pos_k[sk], starts)]
        # (a row of -inf everywhere gives 0, not NaN)
        top = z.detach().amax(dim=-1, keepdim=True)
        dead = top == -float('inf')
        e = torch.exp(z - top.masked_fill(dead, 0))
        p = e / e.sum(dim=-1, keepdim=True).masked_fill(dead, 1)
        outs.append((p @ vs).transpose(0, 1))
    if rows < q.size(0) or not outs:
        outs.append(qa[rows:].masked_fill(never, 0))
    return torch.cat(outs, dim=0).to(q.dtype)


# --------------------------------------------------------------------------
# Layer norm, match log-probabilities
# --------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    s = x if residual is None else x + residual
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    d = s.to(acc) - s.to(acc).mean(dim=-1, keepdim=True)
    y = d / torch.sqrt((d * d).mean(dim=-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(acc)
    if bias is not None:
        y = y + bias.to(acc)
    y = y.to(x.dtype)
    return y if residual is None else (y, s)


def match_log_probs(scores, target, n_cols=None, top=0):
    """``(log_prob, entropy, top_log_prob, top_index)`` of the row softmax
    over the valid columns (see ``ops/logprob.py``)."""
    acc = torch.float64 if scores.dtype == torch.float64 else torch.float32
    V = scores.size(1)
    z = scores.to(acc)
    col = torch.arange(V, device=z.device)
    ninf = torch.full((), -float('inf'), dtype=acc, device=z.device)
    if n_cols is not None:
        z = torch.where(col < n_cols.view(-1, 1), z, ninf)
    top_z = z.detach().amax(dim=-1, keepdim=True)
    empty = top_z == -float('inf')
    m = top_z.masked_fill(empty, 0)
    # (masked entries leave the graph: their gradient is 0)
    live = z != -float('inf')
    d = torch.where(live, z, m) - m
    e = torch.exp(d) * live
    total = e.sum(dim=-1, keepdim=True).masked_fill(empty, 1)
    lp = d - torch.log(total)
    ent = -(e / total * lp).sum(dim=-1)
    given = (target >= 0) & (target < V)
    y = torch.where(given, target, torch.zeros_like(target)).view(-1, 1)
    logp = torch.where(live.gather(1, y), lp.gather(1, y), ninf).view(-1)
    logp = torch.where(given, logp, torch.zeros_like(logp))
    idx = z.detach().sort(dim=-1, descending=True, stable=True)[1][:, :top]
    dead = ~live.gather(1, idx)
    top_lp = lp.detach().gather(1, idx).masked_fill(dead, -float('inf'))
    return logp, ent, top_lp, idx.masked_fill(dead, -1)
