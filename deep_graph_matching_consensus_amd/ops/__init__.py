"""Native op layer: HIP kernels on MI355X, PyTorch oracles on CPU."""
from ._backend import hip_available, host_available, use_hip
from .sparse import SparseOperator, spmm
from .plans import (spline_plan, adjacency_plan, relational_plan,
                    compute_spline_basis, clear_plan_cache)
from .attention import segment_attention
from .logprob import match_log_probs
from .norm import layer_norm
from . import dense, sparse_corr, reference

__all__ = [
    'hip_available', 'host_available', 'use_hip', 'SparseOperator', 'spmm',
    'spline_plan', 'adjacency_plan', 'relational_plan',
    'compute_spline_basis', 'clear_plan_cache', 'segment_attention',
    'match_log_probs', 'layer_norm', 'dense', 'sparse_corr', 'reference',
]
