"""The ragged prefill's plan: every index array of every packed group from its definition, steps whose requests pass a
launch's limits, and what the arrays cost to build on the host."""
import numpy as np
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from kushkash_amd._prefill import ExtendPlan, pack_plan

PAGE = 32


def step(R, seed, new=70, history=400):
    rng = np.random.default_rng(seed)
    q, h = rng.integers(0, new, R), rng.integers(0, history, R) * rng.integers(0, 2, R)
    q[rng.integers(0, R)] += 1
    slots = rng.permutation(R + 5)[:R]
    table = torch.from_numpy(rng.permutation(R * 20).reshape(R, 20).astype(np.int32))
    return q, h, slots, table


def build(q, h, slots, table, budget=None, packed=True):
    return ExtendPlan.build(q, h, slots, table, kv_heads=1, head_dim=64, dtype=torch.bfloat16, packed=packed, budget=budget)


def check(plan, q, h, slots, table):
    """plan against pack_plan of each group's requests, and the write's jobs."""
    assert plan.q_start.tolist() == [0, *np.cumsum(q).tolist()] == plan.q_start_host and plan.history_host == h.tolist()
    jobs = [(r, p) for r in range(len(q)) for p in sorted({(h[r] + i) // PAGE for i in range(q[r])})]
    assert list(zip(plan.job_seq.tolist(), plan.job_page.tolist())) == jobs
    at, host = 0, table.cpu().numpy()
    for g in plan.groups:
        assert g.r0 == at
        at = g.r1
        if not g.packed:
            continue
        sl = slice(g.r0, g.r1)
        p = pack_plan(q[sl], h[sl], slots[sl])
        assert g.key_start == g.cu_k.tolist() == p.key_start.tolist() and g.n_keys == p.key_start[-1]
        assert g.cu_q.tolist() == [0, *np.cumsum(q[sl]).tolist()]
        assert g.page_blk.tolist() == host[sl][p.page_req, p.page_index].tolist() and g.page_dst.tolist() == p.page_dst.tolist()
        assert g.tail_blk.tolist() == host[sl][p.tail_req, h[sl][p.tail_req] // PAGE].tolist()
        assert g.tail_info.tolist() == p.tail_info.reshape(-1).tolist() and g.new_dst.tolist() == p.new_dst.tolist()
        for x in (g.cu_q, g.cu_k, g.page_blk, g.page_dst, g.tail_blk, g.tail_info, g.new_dst):
            assert x.dtype == torch.int32 and x.is_contiguous() and x.device == table.device and x.dim() == 1
        assert (g.max_q, g.max_k, g.has_history) == (q[sl].max(), (q + h)[sl].max(), bool(h[sl].any()))
    assert at == len(q)


@pytest.mark.parametrize("R", [1, 2, 9, 40])
@pytest.mark.parametrize("budget", [None, 0, 60000, 120000, 400000])
@pytest.mark.parametrize("packed", [True, False])
def test_every_group_s_arrays(R, budget, packed):
    for seed in range(3):
        args = step(R, seed)
        plan = build(*args, budget=budget, packed=packed)
        check(plan, *args)
        if not packed:
            assert not any(g.packed for g in plan.groups)


@pytest.mark.parametrize("packed", [True, False])
def test_keys_past_31_bits(packed):
    """Requests whose keys together pass 2^31 where each group's do not (a shared prefix's pages counted for every request)."""
    q, h, slots = np.array([40, 1, 5]), np.array([1 << 30] * 2 + [70]), np.array([2, 0, 1])
    table = torch.zeros(1, (1 << 25) + 3, dtype=torch.int32).expand(3, -1)
    plan = build(q, h, slots, table, budget=1 << 20, packed=packed)
    first = [(0, (1 << 25)), (0, (1 << 25) + 1), (1, 1 << 25), (2, 2)]
    assert list(zip(plan.job_seq.tolist(), plan.job_page.tolist())) == first
    assert [g.packed for g in plan.groups] == [False, False, packed] and plan.history_host == h.tolist()


def test_more_requests_than_a_launch_takes():
    R = 65600
    table = torch.arange(R, dtype=torch.int32)[:, None]
    plan = build(np.ones(R, dtype=np.int64), np.full(R, 3), np.arange(R), table, budget=128 * 2 * 4 * 1000)
    assert plan.job_seq.tolist() == list(range(R)) and not plan.job_page.any()
    assert len(plan.groups) == 66 and plan.groups[1].tail_blk.tolist() == list(range(1000, 2000))
    plan = build(np.ones(R, dtype=np.int64), np.full(R, 3), np.arange(R), table, budget=1 << 30)
    assert plan.job_seq.tolist() == plan.groups[0].tail_blk.tolist() == list(range(R)) and len(plan.groups) == 1


VIEWS = {getattr(torch.ops.aten, name) for name in ("slice", "view", "expand", "alias", "unsqueeze")}


class Ops(TorchDispatchMode):
    """The operations that run under it, views aside: how many, and the most elements one of them makes."""
    count = most = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if func.overloadpacket not in VIEWS:
            self.count += 1
            for x in out if isinstance(out, (tuple, list)) else [out]:
                if isinstance(x, torch.Tensor):
                    self.most = max(self.most, x.numel())
        return out


def test_what_a_plan_costs_on_the_host():
    """A step of many groups takes a few gathers of each on the CPU, not a chain of torch operations (64 groups: 1.8 ms against 9.6)."""
    q, h, slots, table = step(64, 5)
    with Ops() as ops:
        plan = build(q + 1, h, slots, table, budget=120000)
    assert len(plan.groups) > 20 and ops.count <= 8 * len(plan.groups) + 20
