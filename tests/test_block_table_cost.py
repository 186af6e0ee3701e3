"""What a block table costs to build on the host."""
import torch

import kushkash_amd as kk
from test_extend_plan import Ops

PAGE = 32


def test_what_a_block_table_costs_on_the_host():
    """It reads a map at its pages, not whole rows."""
    tokens = torch.arange(7 * 4096, dtype=torch.int32).view(7, 4096)
    req, lens = torch.tensor([6, 0, 3]), torch.tensor([4096, 1, 70])
    with Ops() as ops:
        table, _, _ = kk.block_table(tokens, req, lens, 128)
    assert ops.most <= 3 * 128 and table[0].tolist() == tokens[6, ::PAGE].floor_divide(PAGE).tolist()
    assert table[2].tolist()[:4] == [*(tokens[3, :96:PAGE] // PAGE).tolist(), 0] and table[1].tolist()[:2] == [0, 0]
