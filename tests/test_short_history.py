"""A batch's chunk over a history of one full page (KushCache.attend_chunk): the unpack's index arrays are contiguous."""
import types

import torch

from kushkash_amd import _attention


def test_one_page_of_history_in_a_batch():
    calls = []
    ops = types.SimpleNamespace(dtype=torch.float32, unpack=lambda *a: calls.append(a))
    B, H, T, D, n = 3, 2, 4, 64, 40
    table = torch.arange(B * 5, dtype=torch.int32).view(B, 5)
    k = torch.zeros(B, H, T, D)
    _attention._unpacked_rows(ops, k, k, torch.zeros(15, H, 8, dtype=torch.uint8), table, n, torch.zeros(B, H, 32, D),
                              torch.arange(B, dtype=torch.int32), False)
    page_blk, page_dst, tail_blk, tail_info = calls[0][1:5]
    assert page_blk.tolist() == [0, 5, 10] and page_dst.tolist() == [0, n + T, 2 * (n + T)]
    assert tail_blk.tolist() == [1, 6, 11] and tail_info.view(3, 3)[:, 1].tolist() == [8, 8, 8]
    assert all(x.is_contiguous() for x in (page_blk, page_dst, tail_blk, tail_info))
