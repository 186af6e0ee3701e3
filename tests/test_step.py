"""What surrounds a serving step's attention, on the CPU: map_sizes, step_maps and block_table on the host path against their
definitions, and the refusals that answer before anything is launched."""
import pytest
import torch

import kushkash_amd as kk
from _maps_case import PAGE, check

CASES = [([], []), ([1], [0]), ([0], [0]), ([0], [77]), ([32], [0]), ([33], [31]), ([1, 1, 1], [31, 32, 33]),
         ([5, 0, 70, 1, 32], [0, 40, 100, 63, 64]), ([300, 2, 9], [2000, 900, 0]), ([4] * 70, list(range(0, 700, 10)))]


@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (32, 1), (33, 32), (100, 33), (500, 4), (1 << 30, 0), (5, 5000)])
@pytest.mark.parametrize("new, history", CASES, ids=[str(i) for i in range(len(CASES))])
def test_maps_on_the_host(new, history, window, sinks):
    if new:
        check(kk, torch, new, history, "cpu", window, sinks, seed=len(new))
    else:
        maps = kk.step_maps(*(torch.zeros(0, dtype=torch.int32) for _ in range(3)), torch.zeros(0, 4, dtype=torch.int32),
                            kk.map_sizes(new, history, window=window or None, sinks=sinks))
        assert maps.q_start.tolist() == maps.key_start.tolist() == [0] and maps.slot_map.numel() == 0


@pytest.mark.parametrize("new, history", CASES[1:], ids=[str(i) for i in range(1, len(CASES))])
def test_the_maps_of_a_prefill_step_are_its_plan(new, history):
    """Without a window they are the arrays of the ragged prefill's plan, which numpy builds on the host."""
    from kushkash_amd._prefill import pack_plan
    R = len(new)
    table = torch.arange(1, R * 80 + 1, dtype=torch.int32).view(R, 80)
    slots = torch.arange(R, dtype=torch.int32) + 3
    maps = kk.step_maps(*(torch.tensor(x, dtype=torch.int32) for x in (new, history)), slots, table, kk.map_sizes(new, history))
    plan = pack_plan(new, history, slots.numpy())
    assert maps.key_start.tolist() == plan.key_start.tolist() and maps.page_dst.tolist() == plan.page_dst.tolist()
    assert maps.page_blk.tolist() == table.numpy()[plan.page_req, plan.page_index].tolist()
    assert maps.tail_info.tolist() == plan.tail_info.tolist() and maps.new_dst.tolist() == plan.new_dst.tolist()


def test_sizes():
    s = kk.map_sizes([5, 0, 70], [0, 40, 100])
    assert (s.requests, s.tokens, s.keys, s.pages, s.tails) == (3, 75, 215, 4, 2)
    assert s.writes().numbers == (3, 75, 215, s.jobs, 0, 0, 0, 0)
    w = kk.map_sizes([5], [1000], window=64, sinks=1)
    assert w.keys == 5 + 1000 - PAGE * ((1000 - 63) // PAGE - 1) and w.numbers[-2:] == (64, 1)
    for bad, match in [(lambda: kk.map_sizes([1], [1, 2]), "one length >= 0"), (lambda: kk.map_sizes([-1], [1]), "one length >= 0"),
                       (lambda: kk.map_sizes([1], [1], sinks=2), "sinks are for"), (lambda: kk.map_sizes([1], [1], window=0), "window must"),
                       (lambda: kk.map_sizes([1 << 30, 1 << 30], [0, 0]), "below 2.31"),
                       (lambda: kk.map_sizes([0] * 65537, [0] * 65537), "at most 65536")]:
        with pytest.raises(ValueError, match=match):
            bad()


def test_refusals_of_step_maps():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    size, table = kk.map_sizes([1, 2], [3, 4]), torch.zeros(2, 3, dtype=torch.int32)
    for args, match in [((i32(1), i32(3, 4), i32(0, 1), table), "new_tokens must be"),
                        ((i32(1, 2), i32(3, 4).long(), i32(0, 1), table), "history must be"),
                        ((i32(1, 2), i32(3, 4), i32(0, 9, 1, 9)[::2], table), "slots must be"),
                        ((i32(1, 2), i32(3, 4), i32(0, 1), table[:1]), "a row per request"),
                        ((i32(1, 2), i32(3, 4), i32(0, 1), table.long()), "block_table must be"),
                        ((i32(1, 2), i32(3, 4), i32(0, 1), torch.zeros(3, 2, dtype=torch.int32).t()), "block_table must be")]:
        with pytest.raises(ValueError, match=match):
            kk.step_maps(*args, size)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_block_table_on_the_host(dtype):
    g = torch.Generator().manual_seed(0)
    tokens = torch.randint(0, 1 << 20, (5, 130), generator=g, dtype=torch.int32)
    req, lens = torch.tensor([4, 0, 2, 2, 7, -1], dtype=dtype), torch.tensor([130, 0, 33, 1, 64, 64], dtype=dtype)
    for pages in (0, 1, 3, 5, 9):
        table, sl, slots = kk.block_table(tokens, req, lens, pages)
        for r, (i, n) in enumerate(zip(req.tolist(), lens.tolist())):
            for p in range(pages):
                want = int(tokens[i, PAGE * p]) // PAGE if 0 <= i < 5 and PAGE * p < min(n, 130) else 0
                assert int(table[r, p]) == want
        assert sl.tolist() == lens.tolist() and slots.tolist() == req.tolist()
        assert table.dtype == sl.dtype == slots.dtype == torch.int32
    wide = torch.full((6, 9), 7, dtype=torch.int32)
    got = kk.block_table(tokens, req, lens, 5, out=(wide[:, :5], sl, slots))
    assert torch.equal(got[0], kk.block_table(tokens, req, lens, 5)[0]) and bool((wide[:, 5:] == 7).all())


def test_refusals_of_block_table():
    tokens, r = torch.zeros(5, 64, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    out = torch.zeros(3, 2, dtype=torch.int32), r.clone(), r.clone()
    for args, kw, match in [((tokens.long(), r, r, 2), {}, "req_to_token must be"), ((tokens, r.float(), r, 2), {}, "req must be"),
                            ((tokens, r, r[:2], 2), {}, "seq_lens must be"), ((tokens, r, r, -1), {}, "pages must be"),
                            ((tokens, r, r, 3), dict(out=out), "out.0. must be"), ((tokens, r, r, 2), dict(out=(out[0], r.long(), r)), "out.1. must be"),
                            ((tokens, r, r, 2), dict(out=(out[0][:1].expand(3, 2), r, r)), "rows apart")]:
        with pytest.raises(ValueError, match=match):
            kk.block_table(*args, **kw)


def test_sampling_is_for_the_gpu():
    with pytest.raises(ValueError, match="sample runs on the GPU"):
        kk.sample(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(ValueError, match="logits must be"):
        kk.sample(torch.zeros(2, 5, dtype=torch.float64), torch.zeros(2))
    with pytest.raises(ValueError, match="logits must be"):
        kk.sample(torch.zeros(5, 2).t(), torch.zeros(2))
