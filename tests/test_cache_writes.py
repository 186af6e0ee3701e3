"""The index arrays of a cache's writes: of sequences of one length each, at a cost that does not grow with the batch."""
import pytest
import torch

import kushkash_amd as kk
from test_extend_plan import Ops


@pytest.mark.parametrize("T, n", [(1, 0), (33, 31), (64, 1000), (5, 7)])
@pytest.mark.parametrize("window, sinks", [(None, 0), (40, 4), (32, 33)])
def test_sizes_of_sequences_of_one_length(T, n, window, sinks):
    for B in (1, 3, 70):
        assert kk.map_sizes([T], [n], window=window, sinks=sinks).times(B) == kk.map_sizes([T] * B, [n] * B, window=window, sinks=sinks)


@pytest.mark.parametrize("batch", [1, 40])
@pytest.mark.parametrize("n, T", [(0, 32), (0, 70), (31, 2), (33, 100)])
def test_writes_on_the_host(batch, n, T):
    """The cached tokens are those written, in a few operations whatever the batch is (a write of 33 tokens: 0.14 ms, 0.48 by the
    maps' operations)."""
    c = kk.KushCache(1, 2, 4, 64, batch_size=batch, bits=8, device="cpu", dtype=torch.float32, rotate=False, max_length=200)
    k, v = (torch.randn(batch, 2, n + T, 64, generator=torch.Generator().manual_seed(i)) for i in (1, 2))
    if n:
        c.write(0, k[:, :, :n], v[:, :, :n])
    c.ops.validate = False                                  # (the checks of index values are operations of their own)
    with Ops() as ops:
        c.write(0, k[:, :, n:], v[:, :, n:])
    assert ops.count <= 30 and c.length(0) == n + T
    # 8 bits of a range of at most 10, and fp16 scales: off by less than a tenth
    assert all(float((x - y).abs().max()) < 0.1 for x, y in zip(c.dequantize(0), (k, v)))
    assert c.seq_lens[0].tolist() == [n + T] * batch


@pytest.mark.gpu
def test_a_batch_of_more_sequences_than_a_launch_of_maps_takes():
    B, n, T = 65600, 3, 31
    c = kk.KushCache(1, 1, 1, 64, batch_size=B, bits=8, device="cuda:0", dtype=torch.bfloat16, rotate=False, max_length=64)
    g = torch.Generator(device="cuda:0").manual_seed(1)
    k, v = (torch.randn(B, 1, n + T, 64, generator=g, device="cuda:0", dtype=torch.bfloat16) for _ in range(2))
    for a, b in ((0, n), (n, n + T)):
        c.write(0, k[:, :, a:b], v[:, :, a:b])
    for x, y in zip(c.dequantize(0), (k, v)):
        assert float((x.float() - y.float()).abs().max()) < 0.15       # (and bf16 roundings of values up to 6)
