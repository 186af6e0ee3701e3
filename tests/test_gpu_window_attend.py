"""window_attention on the GPU against the definition in 64 bits.

Tolerance, with u half a step of the type: a weight is rounded once for the product and enters the denominator as rounded, so
an output moves by at most u sum p |v - o| <= 2 u max|v|, and is rounded once itself: u |o| <= u max|v|. Scores are fp32
sums of exact products (2^-24 of them per term: far below u)."""
import pytest
import torch

import kushkash_amd as kk
from _window_case import half_step, rows_reference
from kushkash_amd import _attend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows(T, N, Hk, G, D, dtype, seed, batch=()):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*batch, n, h, D, generator=g).to(dtype) for n, h in ((T, Hk * G), (N, Hk), (N, Hk))]


def check(out, q, k, v, scale, window, sinks):
    ref = rows_reference(q, k, v, scale, window, sinks)
    err = (out.double().cpu() - ref).abs()
    bound = 3 * half_step(q.dtype) * float(v.abs().max())
    assert bool((err <= bound).all()), f"off by {float(err.max() / bound):.2f} of the bound"


@pytest.mark.parametrize("T, N, window, sinks", [
    (1, 1, 1, 0), (1, 1, 5, 3), (3, 3, 1, 0), (3, 3, 1, 1), (64, 64, 10, 2), (65, 65, 64, 0), (150, 150, 33, 65),
    (1, 400, 7, 3), (1, 400, 128, 64), (70, 400, 100, 130), (200, 777, 64, 4), (300, 300, 299, 0), (300, 300, 300, 5),
    (129, 1000, 1 << 30, 0), (33, 1000, 257, 1 << 30)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_length(T, N, window, sinks, D, dtype):
    Hk, G = 2, 3
    q, k, v = rows(T, N, Hk, G, D, dtype, T + N)
    out = kk.window_attention(q[None].to(DEV), k[None].to(DEV), v[None].to(DEV), window=window, sinks=sinks)
    check(out[0], q, k, v, D ** -0.5, window, sinks)


@pytest.mark.parametrize("G", [1, 4, 7, 16])
def test_ragged_rows(G):
    """Packed sequences, some without queries, one token or a whole prompt; offsets given or built."""
    D, Hk, dtype = 128, 2, torch.bfloat16
    spans = [(5, 300), (0, 17), (1, 1), (140, 140), (0, 0), (33, 1200), (1, 90)]
    q, k, v = rows(sum(t for t, _ in spans), sum(n for _, n in spans), Hk, G, D, dtype, G)
    cu = tuple(torch.tensor([0] + [s[i] for s in spans]).cumsum(0).to(torch.int32).to(DEV) for i in (0, 1))
    dev = [x.to(DEV) for x in (q, k, v)]
    for window, sinks in ((50, 0), (64, 70), (1, 1)):
        out = kk.window_attention(*dev, window=window, sinks=sinks, spans=spans, cu=cu)
        assert torch.equal(out, kk.window_attention(*dev, window=window, sinks=sinks, spans=spans))
        a = c = 0
        for t, n in spans:
            if t:
                check(out[a:a + t], q[a:a + t], k[c:c + n], v[c:c + n], D ** -0.5, window, sinks)
            a, c = a + t, c + n


@pytest.mark.parametrize("waves, chunk", [(4, 0), (4, 1), (4, 2), (4, 5), (8, 0), (8, 3)])
@pytest.mark.parametrize("D", [64, 128])
def test_every_split_of_the_keys(waves, chunk, D, monkeypatch):
    """Workgroups of 4 and 8 waves, a row tile's list of key tiles whole or cut anywhere."""
    dtype, Hk, G = torch.float16, 2, 4
    monkeypatch.setattr(_attend, "plan", lambda *a, **k: (waves, chunk))
    _attend._window_plan.cache_clear()
    try:
        for T, N, window, sinks in ((150, 1500, 400, 100), (90, 700, 64, 0), (300, 900, 129, 65)):
            q, k, v = rows(T, N, Hk, G, D, dtype, chunk)
            out = kk.window_attention(q[None].to(DEV), k[None].to(DEV), v[None].to(DEV), window=window, sinks=sinks)
            check(out[0], q, k, v, D ** -0.5, window, sinks)
    finally:
        _attend._window_plan.cache_clear()


def test_batches_strides_and_outputs():
    """Heads-first inputs and outputs, a row slice of a wider buffer, an output in place."""
    dtype, Hk, G, D, T, N = torch.bfloat16, 2, 4, 128, 90, 333
    q, k, v = rows(T, N, Hk, G, D, dtype, 5, batch=(3,))
    heads = [x.transpose(1, 2).contiguous().transpose(1, 2).to(DEV) for x in (q, k, v)]          # [B, rows, H, D] views
    wide = [torch.cat([x, x], -1).to(DEV)[..., :D] for x in (q, k, v)]
    want = kk.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), window=100, sinks=5)
    for b in range(3):
        check(want[b], q[b], k[b], v[b], D ** -0.5, 100, 5)
    for x in (heads, wide):
        assert torch.equal(kk.window_attention(*x, window=100, sinks=5), want)
    for out in (torch.empty_like(want), torch.empty(3, Hk * G, T, D, dtype=dtype, device=DEV).transpose(1, 2),
                torch.empty(3, T, Hk * G, D + 1, dtype=dtype, device=DEV)[..., 1:]):
        got = kk.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), window=100, sinks=5, out=out)
        assert got is out and torch.equal(out, want)


def test_fp32_odd_heads_and_derivatives_take_the_products():
    """What the kernel does not take: fp32 (each product and sum in fp32), head size 48, inputs that ask for derivatives."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, n, h, 48, generator=g) for n, h in ((40, 4), (100, 2), (100, 2)))
    ref = rows_reference(q[0], k[0], v[0], 48 ** -0.5, 30, 2)
    out = kk.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), window=30, sinks=2)
    assert float((out[0].double().cpu() - ref).abs().max()) <= 100 * half_step(torch.float32) * float(v.abs().max())
    q, k, v = (x.to(torch.bfloat16).to(DEV) for x in rows(20, 50, 2, 2, 64, torch.float32, 2, batch=(1,)))
    q.requires_grad_()
    out = kk.window_attention(q, k, v, window=9, sinks=1)
    out.float().square().sum().backward()
    assert q.grad is not None and bool(torch.isfinite(q.grad).all()) and float(q.grad.abs().max()) > 0


def test_infinities_in_keys_that_are_hidden_from_every_row():
    """Keys left out of every row's list of tiles, and hidden scores that are infinite or NaN (finite values): no trace."""
    dtype, D = torch.bfloat16, 128
    q, k, v = rows(40, 900, 2, 4, D, dtype, 8)
    want = kk.window_attention(q[None].to(DEV), k[None].to(DEV), v[None].to(DEV), window=70, sinks=3)
    k[3:900 - 40 - 70] = float("nan")
    k[3:40:2] = float("inf")
    v[64:768] = float("nan")                                               # whole tiles between the sinks and the windows
    got = kk.window_attention(q[None].to(DEV), k[None].to(DEV), v[None].to(DEV), window=70, sinks=3)
    assert torch.equal(got, want)


def test_replays_of_a_captured_call_with_split_keys():
    dtype, D, Hk, G, T, N = torch.bfloat16, 128, 2, 4, 64, 6000
    q, k, v = (x[None].to(DEV) for x in rows(T, N, Hk, G, D, dtype, 9))
    assert _attend._window_plan(q.shape, k.shape, None, _attend.PARTIAL_BYTES, 4000, 4)[3] > 0
    kk.window_attention(q, k, v, window=4000, sinks=4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kk.window_attention(q, k, v, window=4000, sinks=4)
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).to(dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kk.window_attention(q, k, v, window=4000, sinks=4))


def test_refusals():
    q, k, v = (x.to(DEV) for x in rows(4, 9, 2, 2, 64, torch.bfloat16, 3, batch=(1,)))
    ok = dict(window=3, sinks=1)
    for args, kw in (((q, k, v), dict(window=None)), ((q, k, v), dict(window=0)), ((q, k, v), dict(ok, scale=0.0)),
                     ((q, k, v), dict(ok, scale=float("inf"))), ((q[0], k, v), ok), ((q[0], k[0], v[0]), ok),
                     ((q, k.float(), v), ok), ((q, k, v.cpu()), ok), ((q, k, v[:, :5]), ok), ((k, q, q), ok),
                     ((q[:, :, :3], k, v), ok), ((q, k, v), dict(ok, out=torch.empty_like(k))),
                     ((q, k, v), dict(ok, cu=(None, None))), ((q[0], k[0], v[0]), dict(ok, spans=[(4, 8)])),
                     ((q[0], k[0], v[0]), dict(ok, spans=[(5, 4), (-1, 5)])),
                     ((q[0], k[0], v[0]), dict(ok, spans=[(4, 9)], cu=(torch.zeros(1, dtype=torch.int32),) * 2))):
        with pytest.raises(ValueError):
            kk.window_attention(*args, **kw)
    assert kk.window_attention(q[:, :0], k, v, **ok).shape == (1, 0, 4, 64)
