"""Chunks and prompts under a window: their memory, and chunks whose keys are not one per query."""
import pytest
import torch

import kushkash_amd as kk
from kushkash_amd.hf import prompt_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def randn(*shape, seed, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def extra(fn):
    """(fn's result, bytes it allocated at most beyond what was held)"""
    fn()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    out = fn()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - held


@pytest.mark.parametrize("rotate", [False, True])
def test_a_window_that_hides_nothing_keeps_the_chunk_s_memory_bound(rotate):
    """Window and sinks that cover the history and the chunk: the same output as without, in the same memory (history of 134 MB
    in blocks of 16 MB)."""
    H, G, D, n, T = 4, 2, 128, 65536, 64
    plain, wide = (kk.KushCache(1, H, H * G, D, device=DEV, dtype=torch.bfloat16, rotate=rotate, **kw)
                   for kw in (dict(), dict(window=n + T - 4, sinks=4)))
    for a in range(0, n, 8192):
        k, v = randn(1, H, 8192, D, seed=a + 1), randn(1, H, 8192, D, seed=a + 2)
        for c in (plain, wide):
            c.write(0, k, v)
    q, k, v = randn(1, H * G, T, D, seed=3), randn(1, H, T, D, seed=4), randn(1, H, T, D, seed=5)
    want, least = extra(lambda: plain.attend_chunk(0, q, k, v, 1 << 24))
    got, used = extra(lambda: wide.attend_chunk(0, q, k, v, 1 << 24))
    assert torch.equal(got, want) and used <= least + (1 << 20), f"{used >> 20} MiB, {least >> 20} without a window"
    bound = kk.KushCache(1, H, H * G, D, device=DEV, dtype=torch.bfloat16, rotate=rotate, window=n + T - 5, sinks=4)
    assert bound.layer_limit(0) == (n + T - 5, 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window, sinks", [(4096, 0), (3000, 4)])
def test_a_prompt_s_scratch_keeps_within_its_bound(dtype, window, sinks):
    """prompt_attention's block_bytes holds under a window too: scores of 8 x 4,096 x 4,096 in fp32 are 537 MB, partials of split
    bf16 keys up to 268."""
    H, T, D = 8, 4096, 128
    q, k, v = (randn(1, H, T, D, seed=i, dtype=dtype) for i in range(3))
    rows = 4 * q.numel() * (6 if dtype == torch.float32 else 1)              # the output, fp32 rows of a block's keys and values
    out, used = extra(lambda: prompt_attention(q, k, v, D ** -0.5, 1 << 22, window=window, sinks=sinks))
    assert used <= rows + (1 << 24), f"{used >> 20} MiB"
    at = torch.arange(T, device=DEV)
    hidden = (at[None] > at[:, None]) | ((at[None] <= at[:, None] - window) & (at[None] >= sinks))
    for h in (0, 5):
        s = (q[0, h].double() @ k[0, h].double().t().contiguous() * D ** -0.5).masked_fill_(hidden, float("-inf"))
        want = torch.softmax(s, -1) @ v[0, h].double()
        # bf16: the weights' rounding, half a step (2^-8) above the division and below, and the output's; fp32: a score off by
        # 128 roundings of 2^-24 of its terms' sum, below 15, which counts twice in a weight
        off = 3 * 2.0 ** -8 if dtype == torch.bfloat16 else 2 * 128 * 2.0 ** -24 * 15
        assert float((out[0, h].double() - want).abs().max()) <= off * float(v.abs().max())


@pytest.mark.parametrize("window, sinks", [(40, 0), (90, 33), (150, 4)])
@pytest.mark.parametrize("rows", [33, 50])
@pytest.mark.parametrize("batch", [1, 2])
def test_a_chunk_of_more_keys_than_queries(window, sinks, rows, batch):
    """The chunk's queries are the last of its keys: query t stands at history + rows - T + t."""
    T, H, G, D, n = 33, 2, 2, 128, 203
    c = kk.KushCache(1, H, H * G, D, batch_size=batch, bits=8, device=DEV, dtype=torch.bfloat16, rotate=False, window=window, sinks=sinks)
    c.write(0, *(randn(batch, H, n, D, seed=i) for i in (1, 2)))
    hk, hv = (x.double().cpu() for x in c.dequantize(0))
    q, k, v = randn(batch, H * G, T, D, seed=3), randn(batch, H, rows, D, seed=4), randn(batch, H, rows, D, seed=5)
    got = c.attend_chunk(0, q, k, v)
    keys, vals = (torch.cat([h, x.double().cpu()], 2).repeat_interleave(G, 1) for h, x in ((hk, k), (hv, v)))
    p, j = torch.arange(n + rows - T, n + rows)[:, None], torch.arange(n + rows)[None]
    s = (q.double().cpu() @ keys.transpose(2, 3) * c.scale).masked_fill((j > p) | ((j <= p - window) & (j >= sinks)), float("-inf"))
    want = torch.softmax(s, -1) @ vals
    # roundings to bf16 of the history's keys (through scores of about 1) and values, the weights and the output, each at most half
    # a step, evenly spread: 2^-8 / sqrt 3 of the norm
    assert float((got.double().cpu() - want).norm() / want.norm()) < 4 * 2.0 ** -8 / 3 ** 0.5


def test_a_chunk_of_fewer_keys_than_queries_is_refused():
    c = kk.KushCache(1, 2, 4, 128, device=DEV, dtype=torch.bfloat16, window=40)
    c.write(0, randn(1, 2, 100, 128, seed=1), randn(1, 2, 100, 128, seed=2))
    with pytest.raises(ValueError, match="key per query"):
        c.attend_chunk(0, randn(1, 4, 33, 128, seed=3), randn(1, 2, 20, 128, seed=4), randn(1, 2, 20, 128, seed=5))
