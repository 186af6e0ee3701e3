"""The ragged prefill's plan with its block table on the GPU: the same arrays as from the definition, for steps of one and of several
packed groups, and for more requests than a launch takes."""
import numpy as np
import pytest
import torch

from test_extend_plan import build, check, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R", [1, 9, 40])
@pytest.mark.parametrize("budget", [None, 0, 60000, 120000, 400000])
@pytest.mark.parametrize("packed", [True, False])
def test_every_group_s_arrays(R, budget, packed):
    for seed in range(3):
        q, h, slots, table = step(R, seed)
        wide = torch.zeros(R, 33, dtype=torch.int32, device="cuda:0")
        wide[:, :20] = table
        check(build(q, h, slots, wide[:, :20], budget=budget, packed=packed), q, h, slots, wide[:, :20])


def test_keys_past_31_bits():
    q, h, slots = np.array([40, 1, 5]), np.array([1 << 30] * 2 + [70]), np.array([2, 0, 1])
    table = torch.zeros(1, (1 << 25) + 3, dtype=torch.int32, device="cuda:0").expand(3, -1)
    plan = build(q, h, slots, table, budget=1 << 20)
    assert plan.job_seq.tolist() == [0, 0, 1, 2] and plan.job_page.tolist() == [1 << 25, (1 << 25) + 1, 1 << 25, 2]
    assert [g.packed for g in plan.groups] == [False, False, True]


@pytest.mark.parametrize("budget", [128 * 2 * 4 * 1000, 1 << 30])
def test_more_requests_than_a_launch_takes(budget):
    R = 65600
    table = torch.arange(R, dtype=torch.int32, device="cuda:0")[:, None]
    plan = build(np.ones(R, dtype=np.int64), np.full(R, 3), np.arange(R), table, budget=budget)
    assert plan.job_seq.tolist() == list(range(R)) and not plan.job_page.any()
    assert [b for g in plan.groups for b in g.tail_blk.tolist()] == list(range(R))
