"""The sparse product's oracle sums 64-bit inputs in 64 bits."""
import torch

from deep_graph_matching_consensus_amd.ops import reference as ref


def test_spmm_oracle_keeps_64_bit_sums():
    # 1 + 2^-30 - 1: the middle term is lost in 32 bits (unit 2^-24 at 1)
    x = torch.tensor([[1.0], [2.0 ** -30], [-1.0]], dtype=torch.float64)
    row = torch.zeros(3, dtype=torch.int32)
    col = torch.arange(3, dtype=torch.int32)
    out = ref.spmm(row, col, torch.ones(3), 1, x)
    assert out.item() == 2.0 ** -30
    # with bias and self term, rounded once to the output's type
    out = ref.spmm(row, col, torch.ones(3), 1, x,
                   self_x=torch.ones(1, 1, dtype=torch.float64),
                   self_scale=torch.ones((), dtype=torch.float64),
                   bias=-torch.ones(1, dtype=torch.float64))
    assert out.item() == 2.0 ** -30
    # 32-bit inputs keep 32-bit sums
    assert ref.spmm(row, col, torch.ones(3), 1, x.float()).item() == 0.0
