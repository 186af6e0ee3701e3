"""append_decode refused under a window on the CPU: before it appends."""
import pytest
import torch

import kushkash_amd as kk
from kushkash_amd._ops import PAGE


def test_a_refused_append_leaves_the_cache_as_it_was():
    D, H, G, S = 64, 2, 2, 3
    ops = kk.Ops(torch.device("cpu"), D, 4, G, torch.float32)
    cache = torch.zeros(4, H, kk.record_bytes(D, 4), dtype=torch.uint8)
    table, lens = torch.arange(S, dtype=torch.int32)[:, None], torch.tensor([1, 5, 32], dtype=torch.int32)
    tail, slots = torch.zeros(S, H, PAGE, D), torch.arange(S, dtype=torch.int32)
    k, v, q = torch.ones(S, H, D), torch.ones(S, H, D), torch.ones(S, H * G, D)
    out = torch.zeros_like(q)
    with pytest.raises(ValueError, match="window is a GPU extension"):
        ops.append_decode(k, v, q, out, cache, table, lens, slots, tail, 0.1, window=16, sinks=1)
    assert not tail.any() and not cache.any() and not out.any()
    ops.append_decode(k, v, q, out, cache, table, lens, slots, tail, 0.1)
    assert tail.any() and out.any()
