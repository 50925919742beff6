"""Deep Graph Matching Consensus
(API of ``/root/reference/dgmc/models/dgmc.py``).

Public surface kept identical to the reference: constructor
``DGMC(psi_1, psi_2, num_steps, k=-1, detach=False)`` (``dgmc.py:64``),
mutable ``num_steps``/``k``/``detach``/``backend`` attributes, ``forward``
returning ``(S_0, S_L)`` dense ``[sum N_s, N_t]`` tensors or sparse COO
tensors carrying ``__idx__``/``__val__`` (``dgmc.py:228-242``), ``loss``,
``acc``, ``hits_at_k``, ``__include_gt__``, ``reset_parameters`` and the exact
``repr``.  The state-dict schema (``psi_1.*``, ``psi_2.*``, ``mlp.{0,2}.*``)
is unchanged.

What differs is the execution plan (MI355X-first):

* source and target are encoded in ONE call on their disjoint union when the
  encoder allows it (no BatchNorm in training mode) - one large GEMM per layer
  instead of two, half the launches;
* packing between ``[sum N, C]`` and ``[B, N_max, C]`` uses host-precomputed
  index maps (no boolean-mask ``nonzero`` syncs; the reference syncs ~4 times
  per consensus step);
* per-pair softmax/transport and the consensus MLP run as fused HIP kernels
  (factored MLP, no ``[B, N_s, N_t, R]`` tensor);
* the correspondence scores are kept in fp32 even under bf16 autocast (only
  the encoders' GEMMs drop to bf16);
* all random indicators of the L steps are drawn with one ``randn`` call.
"""
import collections
import contextlib

import torch
from torch.nn import Linear, ReLU, Sequential

from ..graph.dense import dense_layout
from ..nn.inits import reset
from ..ops import _backend
from ..ops import dense as dense_ops
from ..ops.gemm import mixed_matmul
from ..ops import relconv as relconv_ops
from ..ops import sparse_corr
from ..ops.logprob import match_log_probs
from ..ops.plans import _IdentityCache
from ..runtime import loopgrad
from ..runtime.cache import forward_cache
from ..runtime.profiling import mark, trace_range
from ..runtime.mode import is_reference_mode
from .encoder import CatParts, StackedEncoder

# FOLD_PROJECTION = False keeps psi_2's final Linear as its own GEMM (tests).
FOLD_PROJECTION = True
# SINKHORN_FUSED = False runs the Sinkhorn consensus loop unfused
# (separate normalisation kernel + batched-GEMM transport).
SINKHORN_FUSED = True

EPS = 1e-8
# Cached sparse-output COO row index tensors (one per (N_s, k, device)).
COO_ROWS_CACHE = 4
_PAIR_CACHE = _IdentityCache(max_entries=8)


class _PackedNLL(torch.autograd.Function):
    """Masked NLL of the dense correspondences (+ Hits@1 count), HIP."""

    @staticmethod
    def forward(ctx, S, y0, y1, mask, mean, with_correct):
        loss, aux = _backend.ops().nll_fwd(S, y0, y1, mask, EPS, mean,
                                           with_correct)
        ctx.save_for_backward(S, y0, y1, mask, aux)
        ctx.mean = mean
        ctx.mark_non_differentiable(aux)
        ctx.set_materialize_grads(False)     # (no zero grad for aux)
        return loss, aux

    @staticmethod
    def backward(ctx, grad, grad_aux):
        if grad is None:
            return (None, ) * 6
        S, y0, y1, mask, aux = ctx.saved_tensors
        dS = _backend.ops().nll_bwd(grad.float().contiguous(), S, y0, y1,
                                    mask, aux, EPS, ctx.mean)
        return dS, None, None, None, None, None


class _SparseNLL(torch.autograd.Function):
    """NLL of the ground truths over top-k candidate lists (+ Hits@1 and
    ground-truth counts), HIP: ``csrc/hip/loss.hip::sparse_nll_*``
    (reference ``dgmc.py:258-266``)."""

    @staticmethod
    def forward(ctx, val, idx, y0, y1, mask, mean):
        loss, aux = _backend.ops().sparse_nll_fwd(val, idx, y0, y1, mask,
                                                  EPS, mean)
        ctx.save_for_backward(val, idx, y0, y1, mask, aux)
        ctx.mean = mean
        ctx.mark_non_differentiable(aux)
        ctx.set_materialize_grads(False)
        return loss, aux

    @staticmethod
    def backward(ctx, grad, grad_aux):
        if grad is None:
            return (None, ) * 6
        val, idx, y0, y1, mask, aux = ctx.saved_tensors
        dval = _backend.ops().sparse_nll_bwd(grad.float().contiguous(), val,
                                             idx, y0, y1, mask, aux, EPS,
                                             ctx.mean)
        return dval, None, None, None, None, None


class _FoldProduct(torch.autograd.Function):
    """``W1 @ W_f`` in fp32 (the folded consensus projection; ``b_f`` rides
    along with an exact zero gradient)."""

    @staticmethod
    def forward(ctx, w1, wf, bf):
        ctx.save_for_backward(w1, wf)
        ctx.bf_like = None if bf is None else (bf.shape, bf.dtype)
        if _backend.use_hip(w1) and w1.dtype == torch.float32 and \
                wf.dtype == torch.float32:
            # fp32 product + its bf16 images W and W^T in one kernel.
            w, wn, wnt = _backend.ops().fold_weights(w1.contiguous(),
                                                     wf.contiguous())
            ctx.mark_non_differentiable(wn, wnt)
            # (no zero-filled gradients for the two bf16 images)
            ctx.set_materialize_grads(False)
            return w, wn, wnt
        with torch.autocast(w1.device.type, enabled=False):
            return w1.float() @ wf.float(), None, None

    @staticmethod
    def backward(ctx, g, _g_wn=None, _g_wnt=None):
        return _FoldProduct._backward(ctx, g)

    @staticmethod
    def _backward(ctx, g):
        w1, wf = ctx.saved_tensors
        if g is None:
            return None, None, None
        g = g.float()
        w1c, wfc, gc = w1.contiguous(), wf.contiguous(), g.contiguous()
        if _backend.use_hip(w1) and w1.dtype == wf.dtype == torch.float32 \
                and wf.size(1) % 4 == 0 and all(
                    t.data_ptr() % 16 == 0 for t in (w1c, wfc, gc)):
            # both products in one launch (relconv.hip::fold_weights_bwd:
            # k-ordered fp32 chains, no library GEMM in the step)
            gw1, gwf = _backend.ops().fold_weights_bwd(w1c, wfc, gc)
            gw1 = gw1 if ctx.needs_input_grad[0] else None
            gwf = gwf if ctx.needs_input_grad[1] else None
        else:
            gw1 = (g @ wf.float().t()).to(w1.dtype) \
                if ctx.needs_input_grad[0] else None
            gwf = (w1.float().t() @ g).to(wf.dtype) \
                if ctx.needs_input_grad[1] else None
        gbf = None
        if ctx.bf_like is not None and ctx.needs_input_grad[2]:
            gbf = g.new_zeros(ctx.bf_like[0], dtype=ctx.bf_like[1])
        return gw1, gwf, gbf


class _RawCandidates(object):
    """Sparse-path candidate scores before the softmax (``DGMC.log_probs``),
    packed ``[sum N_s, k]``."""

    def __init__(self, S_hat_0, S_hat_L, S_idx):
        self.S_hat_0, self.S_hat_L, self.S_idx = S_hat_0, S_hat_L, S_idx


class _RawScores(object):
    """Dense-path scores before the output softmax (``DGMC.objective``,
    ``DGMC.log_probs``)."""

    def __init__(self, S_hat_0, S_hat_L, lay_s, lay_t):
        self.S_hat_0, self.S_hat_L = S_hat_0, S_hat_L
        self.lay_s, self.lay_t = lay_s, lay_t


def _device_type(device):
    return 'cuda' if device.type == 'cuda' else 'cpu'


class _PairGraph(object):
    """Disjoint union of the source and target graph (built once/forward)."""

    def __init__(self, edge_index_s, edge_attr_s, n_s, edge_index_t,
                 edge_attr_t):
        self.n_s = n_s
        self.edge_index = torch.cat(
            [edge_index_s, edge_index_t + n_s], dim=1)
        if edge_attr_s is not None and edge_attr_t is not None:
            self.edge_attr = torch.cat([edge_attr_s, edge_attr_t], dim=0)
        else:
            self.edge_attr = None

    @classmethod
    def from_union(cls, n_s, edge_index, edge_attr):
        pair = cls.__new__(cls)
        pair.n_s, pair.edge_index, pair.edge_attr = n_s, edge_index, edge_attr
        return pair


def register_pair_graph(edge_index_s, edge_attr_s, edge_index_t, edge_attr_t,
                        n_s, edge_index, edge_attr):
    """Provide the disjoint union of a batch's source/target graphs (e.g. a
    static batch whose buffer already holds it) so :meth:`DGMC.forward` does
    not concatenate it.  Keyed on the identity of the four batch tensors."""
    _PAIR_CACHE.put((edge_index_s, edge_attr_s, edge_index_t, edge_attr_t),
                    ('pair', int(n_s)),
                    _PairGraph.from_union(int(n_s), edge_index, edge_attr))


def _cat_rows(a, b):
    """``torch.cat([a, b])`` - or, when ``a`` and ``b`` are consecutive row
    blocks of one contiguous base tensor (static batches), that slice of the
    base (no copy; autograd flows through the base)."""
    base = a._base
    if (base is not None and b._base is base and base.is_contiguous() and
            a.is_contiguous() and b.is_contiguous() and a.dim() >= 1 and
            a.dim() == base.dim() and a.shape[1:] == b.shape[1:] and
            a.shape[1:] == base.shape[1:]):
        row = 1
        for d in a.shape[1:]:
            row *= d
        oa = a.storage_offset() - base.storage_offset()
        ob = b.storage_offset() - base.storage_offset()
        if row > 0 and oa % row == 0 and ob == oa + a.numel():
            i = oa // row
            if i == 0 and a.size(0) + b.size(0) == base.size(0):
                return base      # (no slice: no SliceBackward fill + copy)
            return base[i:i + a.size(0) + b.size(0)]
    return torch.cat([a, b], dim=0)


class DGMC(torch.nn.Module):
    r"""Two-stage deep graph matching (local feature matching followed by
    ``num_steps`` rounds of neighbourhood consensus).

    Args:
        psi_1 (torch.nn.Module): GNN computing node embeddings
            ``psi_1(x, edge_index, edge_attr)`` - or ``psi_1(x, batch)`` for
            a module that ``takes_batch`` (:class:`~..nn.AttentionConv`
            without a position bias).
        psi_2 (torch.nn.Module): GNN validating neighbourhood consensus,
            called likewise; must expose ``in_channels`` (size of the random
            node indicators) and ``out_channels``.
        num_steps (int): number of consensus iterations.
        k (int, optional): sparsity.  ``-1`` keeps dense correspondences.
        detach (bool, optional): stop gradients into ``psi_1``.
        normalization (str, optional): extension - ``'softmax'`` (the
            reference, default) or ``'sinkhorn'`` (dense path only:
            log-domain Sinkhorn with ``sinkhorn_iters`` iterations for
            ``S_0``, every consensus step and ``S_L``).
    """

    def __init__(self, psi_1, psi_2, num_steps, k=-1, detach=False,
                 normalization='softmax', sinkhorn_iters=10):
        super(DGMC, self).__init__()
        assert normalization in ('softmax', 'sinkhorn')
        self.psi_1 = psi_1
        self.psi_2 = psi_2
        self.num_steps = num_steps
        self.k = k
        self.detach = detach
        self.normalization = normalization
        self.sinkhorn_iters = sinkhorn_iters
        self.backend = 'auto'
        R = psi_2.out_channels
        self.mlp = Sequential(Linear(R, R), ReLU(), Linear(R, 1))

    def reset_parameters(self):
        self.psi_1.reset_parameters()
        self.psi_2.reset_parameters()
        reset(self.mlp)

    # ------------------------------------------------------------------
    # Encoding
    # ------------------------------------------------------------------
    @staticmethod
    def _fusable(psi):
        if is_reference_mode():
            return False
        return bool(getattr(psi, 'pair_fusable', False))

    def _encode(self, psi, pair, x_s, x_t, ei_s, ea_s, ei_t, ea_t, batch_s,
                batch_t):
        if pair is not None and self._fusable(psi):
            h = psi(_cat_rows(x_s, x_t), pair.edge_index, pair.edge_attr)
            return h[:pair.n_s], h[pair.n_s:]
        if getattr(psi, 'takes_batch', False):
            return psi(x_s, batch_s), psi(x_t, batch_t)
        return psi(x_s, ei_s, ea_s), psi(x_t, ei_t, ea_t)

    # ------------------------------------------------------------------
    # Sparse helpers
    # ------------------------------------------------------------------
    def __top_k__(self, x_s, x_t):  # pragma: no cover
        r"""Memory-efficient top-k correspondence computation.

        In evaluation mode the GPU filter starts from this model's previous
        candidate lists of the same shape (a persistent warm-start state,
        ``csrc/hip/topk.hip::topk_warm_kernel``): the selected indices do not
        depend on it, only the filter's insertion work does - 1.27 -> 0.85
        ms on the DBP15K shape for repeated queries with unchanged
        embeddings (``tools/bench_topk_warm.py``).  Training steps draw new
        dropout masks in psi_1, which leaves the previous lists too weak a
        bound to pay for the re-score (measured: no net gain), so they
        start cold."""
        warm = None if self.training else self._topk_warm_state(x_s, x_t)
        return sparse_corr.top_k(x_s, x_t, self.k, warm=warm)

    def _topk_warm_state(self, x_s, x_t):
        """Persistent int64 ``[B, N_s, 32]`` candidate state of the top-k
        filter for this shape (-1: cold); allocated outside any capture."""
        if not (_backend.use_hip(x_s) and x_s.dim() == 3):
            return None
        key = (tuple(x_s.shape[:2]), x_t.size(1), str(x_s.device))
        cache = self.__dict__.setdefault('_topk_warm',
                                         collections.OrderedDict())
        st = cache.get(key)
        if st is None:
            if torch.cuda.is_current_stream_capturing():
                return None
            st = cache[key] = torch.full(
                (x_s.size(0), x_s.size(1), 32), -1, dtype=torch.long,
                device=x_s.device)
            while len(cache) > 2:
                cache.popitem(last=False)
        return st

    @staticmethod
    def _include_gt(S_idx, dense_rows, y):
        """Sync-free ground-truth injection: for every GT pair whose target is
        not among the candidates, overwrite the LAST candidate slot."""
        B, N_s, k = S_idx.shape
        row, col = y[0], y[1]
        flat = S_idx.reshape(B * N_s, k)
        pos = dense_rows[row]
        present = (flat[pos] == col.view(-1, 1)).any(dim=-1)
        last = torch.where(present, flat[pos, k - 1], col)
        flat = flat.clone()
        flat[pos, k - 1] = last
        return flat.view(B, N_s, k)

    def __include_gt__(self, S_idx, s_mask, y):
        r"""Includes the ground-truth values in ``y`` into ``S_idx``."""
        dense_rows = s_mask.view(-1).nonzero().view(-1)
        return self._include_gt(S_idx, dense_rows, y)

    def _foldable(self):
        return (FOLD_PROJECTION and not is_reference_mode() and
                isinstance(self.psi_2, StackedEncoder) and self.psi_2.lin and
                isinstance(self.mlp[0], Linear))

    # ------------------------------------------------------------------
    def forward(self, x_s, edge_index_s, edge_attr_s, batch_s, x_t,
                edge_index_t, edge_attr_t, batch_t, y=None):
        r"""Returns initial and refined correspondences ``(S_0, S_L)`` of
        shape ``[batch_size * num_nodes, num_nodes]`` (dense or sparse)."""
        with forward_cache():
            return self._forward(x_s, edge_index_s, edge_attr_s, batch_s, x_t,
                                 edge_index_t, edge_attr_t, batch_t, y)

    def _forward(self, x_s, edge_index_s, edge_attr_s, batch_s, x_t,
                 edge_index_t, edge_attr_t, batch_t, y, raw=False):
        device = x_s.device
        dev_type = _device_type(device)
        outer_autocast = torch.is_autocast_enabled(dev_type)
        outer_dtype = torch.get_autocast_dtype(dev_type)
        pair = None
        if self._fusable(self.psi_1) or self._fusable(self.psi_2):
            # Memoised on tensor identity+version: a static graph (e.g. a
            # KG trained full-batch) keeps its union graph and hence all its
            # cached message-passing plans across steps.
            key = (edge_index_s, edge_attr_s, edge_index_t, edge_attr_t)
            params = ('pair', x_s.size(0))
            pair = _PAIR_CACHE.get(key, params)
            if pair is None:
                pair = _PAIR_CACHE.put(key, params, _PairGraph(
                    edge_index_s, edge_attr_s, x_s.size(0), edge_index_t,
                    edge_attr_t))

        with trace_range('dgmc.psi_1'):
            h_s, h_t = self._encode(self.psi_1, pair, x_s, x_t, edge_index_s,
                                    edge_attr_s, edge_index_t, edge_attr_t,
                                    batch_s, batch_t)
        if self.detach:
            h_s, h_t = h_s.detach(), h_t.detach()

        lay_s = dense_layout(batch_s, h_s.size(0), device)
        lay_t = dense_layout(batch_t, h_t.size(0), device)
        assert lay_s.B == lay_t.B, 'Encountered unequal batch-sizes'
        B, N_s, N_t = lay_s.B, lay_s.N, lay_t.N
        n_s, n_t = lay_s.counts, lay_t.counts
        R_in = self.psi_2.in_channels
        steps = self.num_steps or 0

        # loop_scope: psi_2 / MLP weight gradients of the num_steps uses are
        # accumulated in place (runtime/loopgrad.py) instead of per use.
        with torch.autocast(device_type=dev_type, enabled=False), \
                loopgrad.loop_scope(not is_reference_mode()):
            f32 = torch.float64 if h_s.dtype == torch.float64 \
                else torch.float32
            # Dense path on the GPU: S_hat straight from the packed joint
            # encoder output (one per-pair kernel, no padded copies).
            h_joint = _cat_rows(h_s, h_t) if self.k < 1 else None
            direct = h_joint is not None and h_joint.data_ptr() == \
                h_s.data_ptr() and dense_ops.pair_scores_supported(
                    h_joint, lay_s, lay_t)
            if not direct:
                hs = lay_s.to_dense(h_s.to(f32))
                ht = lay_t.to_dense(h_t.to(f32))
            # Random node indicators for all steps, packed [steps, sum N_s, R]
            # (drawn directly in the encoder GEMM dtype under autocast).
            r_dtype = outer_dtype if (outer_autocast and self.k < 1 and
                                      device.type == 'cuda' and
                                      not is_reference_mode()) else f32
            if steps > 0:
                r_all = torch.randn((steps, lay_s.num_nodes, R_in),
                                    dtype=r_dtype, device=device)

            def refine(r_s, r_t, r_joint=None, features=False):
                """psi_2 on both graphs (packed in/out) under the caller's
                autocast policy; returns (o_s, o_t, o_joint or None).
                ``r_joint`` = ``[r_s; r_t]`` already assembled; ``features``
                skips psi_2's final Linear (folded by the caller)."""
                # features: psi_2's final Linear is folded by the caller; its
                # concatenated features may stay unformed (CatParts, read
                # in place by the consensus projection).
                ctx = (self.psi_2.features_parts() if hasattr(
                    self.psi_2, 'features_parts') else
                    self.psi_2.features_only()) if features else \
                    contextlib.nullcontext()
                with torch.autocast(device_type=dev_type, dtype=outer_dtype,
                                    enabled=outer_autocast), ctx:
                    if pair is not None and self._fusable(self.psi_2):
                        if r_joint is None:
                            r_joint = torch.cat([r_s, r_t], dim=0)
                        else:
                            # [r_s; r_t] from the transport: only the r_t rows
                            # carry a gradient (r_s is a random constant), so
                            # psi_2's first layer skips the r_s input
                            # gradient (ops/slot_gemm.py).
                            r_joint._dgmc_dx_row0 = int(pair.n_s)
                        o = self.psi_2(r_joint, pair.edge_index,
                                       pair.edge_attr)
                        if isinstance(o, CatParts):
                            return None, None, o
                        return o[:pair.n_s], o[pair.n_s:], o
                    o_s, o_t = self._encode(
                        self.psi_2, None, r_s, r_t, edge_index_s, edge_attr_s,
                        edge_index_t, edge_attr_t, batch_s, batch_t)
                    return o_s, o_t, None

            if self.k < 1 and self.normalization == 'sinkhorn':
                # ---------- dense variant, Sinkhorn (extension) ---------- #
                if direct:
                    S_hat = dense_ops.pair_scores(h_joint, h_s.size(0),
                                                  lay_s, lay_t)
                else:
                    S_hat = hs @ ht.transpose(-1, -2)
                return self._dense_sinkhorn(S_hat, r_all, steps, lay_s,
                                            lay_t, refine, pair)
            assert self.normalization == 'softmax', \
                'Sinkhorn normalisation is only defined for k=-1 (dense)'
            if self.k < 1:
                # ------------------ dense variant -------------------- #
                # raw: the caller (objective) fuses softmax + NLL on the
                # scores themselves; the probabilities are never formed.
                two = False
                if direct:
                    # Raw objective + consensus steps: S_hat_0 has two
                    # consumers - one handle each (no autograd add).
                    two = raw and steps > 0 and torch.is_grad_enabled()
                    S_hat = dense_ops.pair_scores(h_joint, h_s.size(0),
                                                  lay_s, lay_t, two=two)
                else:
                    S_hat = hs @ ht.transpose(-1, -2)        # [B, N_s, N_t]
                if two:
                    S_hat_0, S_hat = S_hat
                else:
                    S_hat_0 = S_hat
                raw = raw == 'scores' or (
                    raw and dense_ops.softmax_nll_supported(S_hat, lay_s))
                S_0 = None if raw else \
                    dense_ops.masked_softmax_packed(S_hat, lay_s, lay_t)
                # Fused pair encoding: the transport kernel writes r_t
                # straight into psi_2's joint input [r_s; r_t] (no cat).
                joint = steps > 0 and pair is not None and \
                    self._fusable(self.psi_2) and \
                    dense_ops.transport_joint_supported(S_hat, lay_s, lay_t)
                # psi_2's final Linear folded into the MLP's first layer:
                # P_i - Q_j = (o_s,i - o_t,j) W1^T with o = h W_f^T + b_f, so
                # [P; Q] = h (W1 W_f)^T - b_f cancels in the difference.  One
                # node-level GEMM per step instead of two (forward and
                # backward); the fold's weight gradient flows through the
                # tiny W1 W_f product once per step.
                fold = self._dense_fold(steps) if joint else None
                # psi_2's first conv on the bf16x6 slot path: the transport
                # kernels also write the joint's operand planes.
                planes = joint and steps > 0 and hasattr(
                    self.psi_2, 'takes_x6_planes') and \
                    self.psi_2.takes_x6_planes(r_all[0])
                pending = None    # (joint, S_hat) from a fused step boundary
                for step in range(steps):
                    mark('dgmc.consensus_step')
                    r_s = r_all[step]
                    if pending is not None:
                        r_joint, S_hat = pending
                        pending = None
                        o_s, o_t, o = refine(None, None, r_joint,
                                             features=fold is not None)
                    elif joint and S_hat.requires_grad and \
                            torch.is_grad_enabled():
                        # S_hat feeds the transport AND the update: the
                        # update reads it through the transport's alias, so
                        # both gradients meet in the transport backward.
                        r_joint, S_hat = dense_ops.softmax_transport_joint(
                            S_hat, r_s, lay_s, lay_t, passthrough=True,
                            planes=planes)
                        o_s, o_t, o = refine(None, None, r_joint,
                                             features=fold is not None)
                    elif joint:
                        r_joint = dense_ops.softmax_transport_joint(
                            S_hat, r_s, lay_s, lay_t, planes=planes)
                        o_s, o_t, o = refine(None, None, r_joint,
                                             features=fold is not None)
                    else:
                        r_t = dense_ops.softmax_transport(S_hat, r_s, lay_s,
                                                          lay_t)
                        o_s, o_t, o = refine(r_s, r_t)
                    # With the fold, the consensus update also runs the next
                    # step's softmax transport (one fused per-pair kernel).
                    nxt = r_all[step + 1] if (fold is not None and joint and
                                              step + 1 < steps) else None
                    res = dense_ops.consensus_update(
                        S_hat, o_s, o_t, self.mlp, lay_s, lay_t, o_joint=o,
                        w1_fold=fold, next_r_s=nxt, planes=planes)
                    if isinstance(res, tuple):
                        pending = res
                    else:
                        S_hat = res
                if raw:
                    return _RawScores(S_hat_0, S_hat, lay_s, lay_t)
                S_L = dense_ops.masked_softmax_packed(S_hat, lay_s, lay_t)
                return S_0, S_L

            # ------------------- sparse variant ---------------------- #
            with trace_range('dgmc.top_k'):
                S_idx = self.__top_k__(hs, ht)                # [B, N_s, k]
            if self.training and y is not None:
                kr = min(self.k, N_t - self.k)
                if _backend.use_hip(S_idx):
                    # K12 in two launches: candidates + negatives, then the
                    # ground-truth patch (csrc/hip/candidates.hip).
                    S_idx = _backend.ops().train_candidates(
                        S_idx.contiguous(), N_t, max(kr, 0),
                        (y[0] if lay_s.identity else lay_s.index[y[0]])
                        .long().contiguous(), y[1].long().contiguous())
                else:
                    S_rnd_idx = torch.randint(N_t, (B, N_s, kr),
                                              dtype=torch.long, device=device)
                    S_idx = torch.cat([S_idx, S_rnd_idx], dim=-1)
                    S_idx = self._include_gt(S_idx, lay_s.index, y)
            k = S_idx.size(-1)
            # CSR/CSC of the candidate set, shared by every op of the loop.
            cand = sparse_corr.CandidateGraph(S_idx, N_t) \
                if device.type == 'cuda' and not is_reference_mode() else None

            S_hat = sparse_corr.gather_dot(hs, ht, S_idx, cand)  # [B,N_s,k]
            S_hat_0 = S_hat
            S = S_hat.softmax(dim=-1)      # S_0 and step 0's S (one softmax)
            S_0 = lay_s.to_sparse(S)
            # psi_2's final Linear folded into the MLP's first layer, as in
            # the dense path: [P; Q] = feat (W1 W_f)^T on psi_2's joint
            # features (b_f cancels in P_i - Q_idx) - one node GEMM per step
            # instead of three (final Linear, P, Q), forward and backward.
            fold_w = rel = None
            if steps > 0 and cand is not None and pair is not None and \
                    self._fusable(self.psi_2) and self._foldable() and \
                    lay_s.identity and lay_t.identity:
                # RelCNN psi_2 of the DBP15K config: the whole encoder +
                # folded projection as fused HIP kernels (ops/relconv.py).
                if relconv_ops.supported(self.psi_2, self.psi_2.final,
                                         self.mlp[0]):
                    rel = relconv_ops.rel_plan(pair.edge_index,
                                               lay_s.num_nodes +
                                               lay_t.num_nodes)
                if rel is None:
                    fold_w = _FoldProduct.apply(self.mlp[0].weight,
                                                self.psi_2.final.weight,
                                                self.psi_2.final.bias)[0]
            # The consensus kernel also emits softmax(S_hat') - the next
            # step's S and finally S_L (dgmc.py:205,225) - and runs its
            # backward: no separate softmax kernels nor gradient add.
            fused_soft = (fold_w is not None or rel is not None) and \
                sparse_corr.soft_fusable(k, self.mlp[0].weight.size(0))
            for step in range(steps):
                if step > 0 and not fused_soft:
                    S = S_hat.softmax(dim=-1)
                r_s = r_all[step]
                r_t = sparse_corr.sparse_transport(
                    S, lay_s.to_dense(r_s), S_idx, N_t, cand)
                if rel is not None:
                    PQ = relconv_ops.psi2_fold(
                        self.psi_2, self.mlp[0].weight, rel, r_s,
                        r_t.reshape(-1, r_t.size(-1)),
                        (id(self.psi_2), rel.N))
                    res = sparse_corr.consensus_update_pq(
                        S_hat, PQ, pair.n_s, self.mlp, cand,
                        with_prob=fused_soft)
                    if fused_soft:
                        S_hat, S = res
                    else:
                        S_hat = res
                    continue
                if fold_w is not None:
                    _, _, feat = refine(r_s, lay_t.to_sparse(r_t),
                                        features=True)
                    # (split-K weight gradient, accumulated over the loop's
                    # steps into one long-K product: runtime/loopgrad.py)
                    PQ = mixed_matmul(feat.to(f32), fold_w.t(), fold_w.t(),
                                      loop_key=('sparse_fold',
                                                id(self.mlp[0].weight)))
                    res = sparse_corr.consensus_update_pq(
                        S_hat, PQ, pair.n_s, self.mlp, cand,
                        with_prob=fused_soft)
                    if fused_soft:
                        S_hat, S = res
                    else:
                        S_hat = res
                    continue
                o_s, o_t, _ = refine(r_s, lay_t.to_sparse(r_t))
                S_hat = sparse_corr.consensus_update(
                    S_hat, lay_s.to_dense(o_s.to(f32)),
                    lay_t.to_dense(o_t.to(f32)), S_idx, self.mlp, cand)
            if raw == 'scores':
                return _RawCandidates(lay_s.to_sparse(S_hat_0),
                                      lay_s.to_sparse(S_hat),
                                      lay_s.to_sparse(S_idx))
            S_L = lay_s.to_sparse(S if (fused_soft or steps == 0) else
                                  S_hat.softmax(dim=-1))
            S_idx = lay_s.to_sparse(S_idx)

        # COO row indices are a function of (N_s, k) only: built once and
        # kept (one stack kernel per forward instead of arange + copy + cat).
        # A small LRU: variable-size batches (eager sparse training) must
        # not keep one [N_s * k] tensor per distinct node count alive.
        key = (x_s.size(0), k, str(device))
        cache = self.__dict__.setdefault('_coo_rows',
                                         collections.OrderedDict())
        row = cache.get(key)
        if row is not None:
            cache.move_to_end(key)
        else:
            row = torch.arange(x_s.size(0), device=device).view(-1, 1)
            row = row.expand(-1, k).reshape(-1)
            if not (device.type == 'cuda' and
                    torch.cuda.is_current_stream_capturing()):
                cache[key] = row            # (never a graph-pool tensor)
                while len(cache) > COO_ROWS_CACHE:
                    cache.popitem(last=False)
        idx = torch.stack([row, S_idx.reshape(-1)], dim=0)
        size = torch.Size([x_s.size(0), N_t])
        out = []
        for val in (S_0, S_L):
            S = torch.sparse_coo_tensor(idx, val.reshape(-1), size,
                                        requires_grad=val.requires_grad)
            S.__idx__ = S_idx
            S.__val__ = val
            out.append(S)
        return tuple(out)

    def _dense_fold(self, steps):
        """psi_2's final Linear folded into the MLP's first layer (dense
        path): ``(W1 W_f)^T``, its bf16 operand images, loop key, uses - or
        None when not foldable."""
        if not self._foldable():
            return None
        # (b_f's exact gradient is zero; it stays in the graph for
        # autograd.grad / DDP.)
        lp = {}
        w_fold, wn, wnt = _FoldProduct.apply(
            self.mlp[0].weight, self.psi_2.final.weight,
            self.psi_2.final.bias)
        if wn is not None:
            # bf16 operand images from the same kernel
            # (ops/dense.py::cat_matmul reads them here).
            lp = {'n': wn, 'nt': wnt}
        return (w_fold.t(), lp, ('fold', id(self.mlp[0].weight)), steps)

    def _dense_sinkhorn(self, S_hat, r_all, steps, lay_s, lay_t, refine,
                        pair):
        """Dense path with Sinkhorn normalisation (opt-in extension): the
        same consensus loop with a masked log-domain Sinkhorn (HIP kernel
        per pair, ``csrc/hip/sinkhorn.hip``) in place of the row softmax.

        On the GPU each step's normalisation and transport ``r_t = S^T r_s``
        run as ONE per-pair kernel writing psi_2's joint input ``[r_s; r_t]``
        (step 0's also emits ``S_0``), whose backward forms
        ``dL/dS = r_s g_t^T`` itself; psi_2's final Linear is folded into the
        consensus MLP as on the softmax path.  Elsewhere: the normalisation
        kernel / oracle and a batched-GEMM transport."""
        iters = self.sinkhorn_iters

        def norm(S_hat):
            return dense_ops.masked_sinkhorn(S_hat, lay_s, lay_t, iters)

        fused = (SINKHORN_FUSED and steps > 0 and pair is not None and
                 self._fusable(self.psi_2) and not is_reference_mode() and
                 r_all.dtype == torch.float32 and
                 dense_ops.sinkhorn_transport_supported(S_hat, r_all[0],
                                                        lay_s, lay_t))
        if not fused:
            S = norm(S_hat)
            S_0 = lay_s.to_sparse(S)
            for step in range(steps):
                r_s = r_all[step]
                if step > 0:
                    S = norm(S_hat)
                r_t = lay_t.to_sparse(S.transpose(-1, -2) @
                                      lay_s.to_dense(r_s.to(S.dtype)))
                o_s, o_t, o = refine(r_s, r_t.to(r_s.dtype))
                S_hat = dense_ops.consensus_update(S_hat, o_s, o_t, self.mlp,
                                                   lay_s, lay_t, o_joint=o)
            return S_0, lay_s.to_sparse(norm(S_hat))

        fold = self._dense_fold(steps)
        P0 = None
        for step in range(steps):
            mark('dgmc.consensus_step')
            grad = S_hat.requires_grad and torch.is_grad_enabled()
            res = dense_ops.sinkhorn_transport_joint(
                S_hat, r_all[step], lay_s, lay_t, iters,
                with_prob=step == 0, passthrough=grad)
            if step == 0 and grad:
                r_joint, P0, S_hat = res
            elif step == 0:
                r_joint, P0 = res
            elif grad:
                r_joint, S_hat = res
            else:
                r_joint = res
            o_s, o_t, o = refine(None, None, r_joint,
                                 features=fold is not None)
            S_hat = dense_ops.consensus_update(
                S_hat, o_s, o_t, self.mlp, lay_s, lay_t, o_joint=o,
                w1_fold=fold)
        return lay_s.to_sparse(P0), lay_s.to_sparse(norm(S_hat))

    # ------------------------------------------------------------------
    # Objectives and metrics (dgmc.py:246-311)
    # ------------------------------------------------------------------
    def objective(self, x_s, edge_index_s, edge_attr_s, batch_s, x_t,
                  edge_index_t, edge_attr_t, batch_t, y_col, mask=None,
                  stats=None):
        r"""The reference drivers' training objective (``pascal.py:67-72``):
        ``NLL(S_0) + NLL(S_L)`` (``NLL(S_0)`` alone when ``num_steps`` is 0)
        for ground truth ``y = (arange(sum N_s), y_col)``, plus the Hits@1
        count of ``S_L``.  Returns ``(loss, count, correct)`` as device
        tensors (``mask`` selects the valid ground truths of a padded
        batch).  ``stats`` (optional fp64 device tensor): ``+= [loss,
        correct, count]`` - folded into the loss kernel on the fused path;
        callers check :attr:`last_stats_fused` to know whether it was.

        On the GPU's dense path the row softmax, NLL and arg-max run as ONE
        fused kernel on the raw scores per output (``softmax_nll``), whose
        backward writes the score gradient directly - the packed
        probabilities are never materialised.  Elsewhere this is
        ``forward`` + :meth:`loss_stats` / :meth:`loss`."""
        with forward_cache():
            out = self._forward(x_s, edge_index_s, edge_attr_s, batch_s, x_t,
                                edge_index_t, edge_attr_t, batch_t, None,
                                raw=True)
        self.last_stats_fused = False
        if isinstance(out, _RawScores):
            y_col = y_col.contiguous()
            # NLL(S_L) + NLL(S_0) (+ the running stats) in one launch + fold.
            loss, aux = dense_ops.softmax_nll(
                out.S_hat_L, out.lay_s, out.lay_t, y_col, mask, EPS,
                S_hat2=out.S_hat_0 if self.num_steps else None, stats=stats)
            self.last_stats_fused = stats is not None
            return loss, aux[0], aux[1]
        S_0, S_L = out
        rows = torch.arange(y_col.numel(), device=y_col.device)
        y = torch.stack([rows, y_col], dim=0)
        if self.num_steps:
            loss_L, count, correct = self.loss_stats(S_L, y, mask)
            return loss_L + self.loss(S_0, y, mask=mask), count, correct
        return self.loss_stats(S_0, y, mask)

    def log_probs(self, x_s, edge_index_s, edge_attr_s, batch_s, x_t,
                  edge_index_t, edge_attr_t, batch_t, y_col=None, top=0,
                  y=None):
        r"""How sure the model is: log-probabilities of the given matches,
        the rows' entropies and the best alternatives, for the initial and
        the refined correspondences (an extension; inputs as in
        :meth:`forward`).

        They are computed from the scores in one pass
        (:func:`~..ops.logprob.match_log_probs`): the probabilities of
        :meth:`forward` are never formed, and a ``log`` of one that has
        underflowed is not taken.

        Args:
            y_col (Tensor, optional): int64 ``[sum N_s]`` given target of
                every source row (a target-graph column, as in
                :meth:`objective`), -1 for none.
            top (int): number of alternatives per row (sparse models: of the
                candidates).
            y (Tensor, optional): ground truth ``[2, num_pairs]`` as in
                :meth:`forward`: in training a sparse model's candidates then
                hold it and random negatives.  Without it they are the best
                ``k`` alone, and a given match outside of them is ``-inf``
                and has no gradient - a loss on it needs ``y``.

        Returns ``(first, last)``, two
        :class:`~..ops.logprob.MatchLogProbs`.  Sparse models: a given match
        that is not among the row's candidates has ``-inf``."""
        if self.normalization != 'softmax':
            raise ValueError('log_probs needs the softmax normalization')
        with forward_cache():
            out = self._forward(x_s, edge_index_s, edge_attr_s, batch_s, x_t,
                                edge_index_t, edge_attr_t, batch_t, y,
                                raw='scores')
        if y_col is None:
            y_col = torch.full((x_s.size(0), ), -1, dtype=torch.long,
                               device=x_s.device)
        if isinstance(out, _RawScores):
            lay_s, lay_t = out.lay_s, out.lay_t
            # valid columns of every packed row (padding rows: graph B, none)
            counts = torch.cat([lay_t.counts, lay_t.counts.new_zeros(1)])
            n_cols = counts[lay_s.index // lay_s.N].to(torch.int32)
            return tuple(match_log_probs(lay_s.to_sparse(S), y_col, n_cols,
                                         top)
                         for S in (out.S_hat_0, out.S_hat_L))
        hit = (out.S_idx == y_col.view(-1, 1)) & (y_col.view(-1, 1) >= 0)
        found = hit.any(dim=-1)
        slot = torch.where(found, hit.to(torch.int8).argmax(dim=-1), -1)
        absent = (y_col >= 0) & ~found
        res = []
        for S in (out.S_hat_0, out.S_hat_L):
            r = match_log_probs(S, slot, top=top)
            col = out.S_idx.gather(1, r.top_index.clamp(min=0))
            res.append(r._replace(
                log_prob=r.log_prob.masked_fill(absent, -float('inf')),
                top_index=torch.where(r.top_index < 0, r.top_index, col)))
        return tuple(res)

    def loss(self, S, y, reduction='mean', mask=None):
        r"""Negative log-likelihood of the ground-truth correspondences.

        Dense: ``-log(S[y0, y1] + eps)``.  Sparse: every candidate slot of
        row ``y0`` holding target ``y1`` contributes (ground truths missing
        from the candidates are dropped, duplicates count twice - as in
        ``dgmc.py:263-265``), evaluated without a host sync.

        ``mask`` (extension): boolean ``[num_gt]`` selecting the valid ground
        truths of a padded static batch; ``'mean'`` then averages over them.
        """
        assert reduction in ['none', 'mean', 'sum']
        if self._fused_nll_ok(S, y, reduction, mask):
            return _PackedNLL.apply(S, y[0].contiguous(), y[1].contiguous(),
                                    mask, reduction == 'mean', False)[0]
        if self._fused_sparse_nll_ok(S, y, reduction, mask):
            return _SparseNLL.apply(S.__val__, S.__idx__, y[0].contiguous(),
                                    y[1].contiguous(), mask,
                                    reduction == 'mean')[0]
        if not S.is_sparse:
            nll = -torch.log(S[y[0], y[1]] + EPS)
            weight = mask
        else:
            assert S.__idx__ is not None and S.__val__ is not None
            hit = S.__idx__[y[0]] == y[1].view(-1, 1)          # [G, k]
            if mask is not None:
                hit = hit & mask.view(-1, 1)
            if reduction == 'none':
                return -torch.log(S.__val__[y[0]][hit] + EPS)
            nll = -torch.log(S.__val__[y[0]] + EPS)
            weight = hit
        if weight is not None:
            nll = nll * weight
            if reduction == 'mean':
                return nll.sum() / weight.sum().clamp(min=1)
        if reduction == 'none':
            return nll
        return nll.mean() if reduction == 'mean' else nll.sum()

    @staticmethod
    def _fused_nll_ok(S, y, reduction, mask):
        return (not S.is_sparse and reduction != 'none' and S.dim() == 2 and
                S.dtype == torch.float32 and S.is_contiguous() and
                y.dtype == torch.long and
                (mask is None or mask.dtype == torch.bool) and
                not is_reference_mode() and _backend.use_hip(S))

    @staticmethod
    def _fused_sparse_nll_ok(S, y, reduction, mask):
        if not (S.is_sparse and reduction != 'none'):
            return False
        val, idx = getattr(S, '__val__', None), getattr(S, '__idx__', None)
        return (val is not None and idx is not None and val.dim() == 2 and
                val.dtype == torch.float32 and val.is_contiguous() and
                idx.dtype == torch.long and idx.is_contiguous() and
                idx.shape == val.shape and y.dtype == torch.long and
                (mask is None or mask.dtype == torch.bool) and
                not is_reference_mode() and _backend.use_hip(val))

    def loss_stats(self, S, y, mask=None):
        """``(loss (mean), ground-truth count, correct top-1 count)`` as device
        tensors - :meth:`loss` and :meth:`correct` in one pass (one fused
        kernel on the GPU, no host sync)."""
        if self._fused_nll_ok(S, y, 'mean', mask):
            loss, aux = _PackedNLL.apply(S, y[0].contiguous(),
                                         y[1].contiguous(), mask, True, True)
            return loss, aux[0], aux[1]
        if self._fused_sparse_nll_ok(S, y, 'mean', mask):
            loss, aux = _SparseNLL.apply(S.__val__, S.__idx__,
                                         y[0].contiguous(), y[1].contiguous(),
                                         mask, True)
            return loss, aux[2], aux[1]
        loss = self.loss(S, y, mask=mask)
        count = (torch.full((), y.size(1), dtype=torch.float32,
                            device=S.device) if mask is None else
                 mask.sum().float())
        return loss, count, self.correct(S.detach(), y, mask).float()

    @staticmethod
    def _predict(S, rows):
        if not S.is_sparse:
            return S[rows].argmax(dim=-1)
        assert S.__idx__ is not None and S.__val__ is not None
        return S.__idx__[rows, S.__val__[rows].argmax(dim=-1)]

    def correct(self, S, y, mask=None):
        """Device tensor with the number of correct top-1 predictions."""
        hit = self._predict(S, y[0]) == y[1]
        if mask is not None:
            hit = hit & mask
        return hit.sum()

    def acc(self, S, y, reduction='mean'):
        r"""Top-1 accuracy (Python number, like the reference)."""
        assert reduction in ['mean', 'sum']
        correct = self.correct(S, y).item()
        return correct / y.size(1) if reduction == 'mean' else correct

    def hits_count(self, k, S, y):
        r"""Device tensor: number of ground truths ranked within the top
        ``k`` (``dgmc.py:290-311``) - without sorting.  The ground truth's
        rank is the number of scores above it plus the equal scores at a
        lower index (the order of a stable descending sort), so one
        elementwise pass per row replaces the reference's full ``argsort``;
        sparse duplicates of the ground truth count once per slot, as in the
        reference's ``(pred == y).sum()``."""
        if not S.is_sparse:
            rows = S[y[0]]                                   # [G, N_t]
            v = rows.gather(1, y[1].view(-1, 1))
            col = torch.arange(rows.size(1), device=rows.device)
            rank = (rows > v).sum(1) + ((rows == v) &
                                        (col < y[1].view(-1, 1))).sum(1)
            return (rank < k).sum()
        assert S.__idx__ is not None and S.__val__ is not None
        idx, val = S.__idx__[y[0]], S.__val__[y[0]]          # [G, k']
        slot = torch.arange(val.size(1), device=val.device)
        # rank[g, c] of candidate slot c among its row's values
        vc = val.unsqueeze(2)                                # [G, k', 1]
        vo = val.unsqueeze(1)                                # [G, 1, k']
        rank = (vo > vc).sum(2) + ((vo == vc) &
                                   (slot.view(1, 1, -1) <
                                    slot.view(1, -1, 1))).sum(2)
        hit = (idx == y[1].view(-1, 1)) & (rank < k)
        return hit.sum()

    def hits_at_k(self, k, S, y, reduction='mean'):
        r"""Fraction of ground truths ranked within the top ``k``."""
        assert reduction in ['mean', 'sum']
        correct = self.hits_count(k, S, y).item()
        return correct / y.size(1) if reduction == 'mean' else correct

    def __repr__(self):
        return ('{}(\n'
                '    psi_1={},\n'
                '    psi_2={},\n'
                '    num_steps={}, k={}\n)').format(type(self).__name__,
                                                    self.psi_1, self.psi_2,
                                                    self.num_steps, self.k)
