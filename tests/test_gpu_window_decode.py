"""Ops.decode and append_decode under a window on the GPU, against the definition in 64 bits.

Tolerance. A weight goes into the product as P' = fp16(e v_scale) and its sum with the same rounding for every part of
a value's code, so an output is off by at most the relative error 2^-11 of each weighted value, and by the
same once more where the weights' sum is not rounded: 2 * 2^-11 of the largest |value| seen. Scores carry fp16 pairs (2^-22
of sums below 2^7: 2^-15 in the exponent, 2^-14 of a value, within a quarter of the first term). Then the output's own
rounding, half a step of its type."""
import pytest
import torch

import kushkash_amd as kk
from _window_case import PAGE, decode_reference, half_step, paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LENS = [0, 1, 31, 32, 33, 64, 95, 200, 331, 1025]


def run(c, q, D, bits, G, dtype, window, sinks, splits=1, waves=None, rot=False, k=None, v=None):
    ops = kk.Ops(torch.device(DEV), D, bits, G, dtype)
    S, H = q.shape[0], c["tail"].shape[1]
    out = torch.full_like(q, float("nan"))
    work = torch.empty(S * H * splits * G * (D + 2), dtype=torch.float32, device=DEV)
    args = (q, out, c["records"], c["table"], c["lens"], c["tidx"], c["tail"], D ** -0.5, splits, work)
    print(f"D={D} bits={bits} G={G} {dtype} window={window} sinks={sinks} splits={splits} waves={waves} rot={rot}", flush=True)
    kw = dict(waves=waves, rot=rot, window=window, sinks=sinks)
    if k is None:
        ops.decode(*args, **kw)
    else:
        ops.append_decode(k, v, *args, **kw)
    torch.cuda.synchronize()
    return out


def check(out, ref, most, dtype):
    bound = 2.5 * 2.0 ** -11 * most + half_step(dtype) * (ref.abs() + 2.0 ** -9 * most)
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), f"off by {float((err / bound).max()):.2f} of the bound"


def case(D=128, bits=4, G=4, H=2, dtype=torch.bfloat16, lens=LENS, seed=0):
    c = paged(lens, D, bits, H, dtype, seed, DEV)
    g = torch.Generator().manual_seed(seed + 1)
    return c, torch.randn(len(lens), H * G, D, generator=g).to(dtype).to(DEV)


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (2, 33), (31, 0), (32, 0), (33, 1), (64, 32), (100, 4), (100, 70),
                                           (300, 500), (2000, 0), (2000, 40), (1 << 30, 1 << 30)])
@pytest.mark.parametrize("splits", [1, 3])
def test_windows_and_sinks(window, sinks, splits):
    c, q = case()
    ref, most = decode_reference(q, c, 128, 4, 4, 128 ** -0.5, window, sinks)
    check(run(c, q, 128, 4, 4, torch.bfloat16, window, sinks, splits), ref, most, torch.bfloat16)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("G, dtype", [(1, torch.float16), (7, torch.bfloat16), (12, torch.float32), (20, torch.bfloat16)])
@pytest.mark.parametrize("waves", [2, 4])
def test_formats(D, bits, G, dtype, waves):
    """Head sizes, record formats, one and two page streams and head chunks, every dtype."""
    c, q = case(D, bits, G, 2 if G < 20 else 1, dtype, seed=3)
    ref, most = decode_reference(q, c, D, bits, G, D ** -0.5, 90, 5)
    check(run(c, q, D, bits, G, dtype, 90, 5, splits=2, waves=waves), ref, most, dtype)


@pytest.mark.parametrize("splits", [1, 7])
def test_a_long_table_and_several_windows_of_ids(splits):
    """Over 1,024 pages: the block ids are gathered behind the length, and a split's list takes more than one table."""
    c, q = case(64, 4, 4, 1, torch.float16, lens=[40000, 36001], seed=4)
    for window, sinks in ((35000, 50), (70, 33), (39999, 0)):
        ref, most = decode_reference(q, c, 64, 4, 4, 64 ** -0.5, window, sinks)
        check(run(c, q, 64, 4, 4, torch.float16, window, sinks, splits), ref, most, torch.float16)


@pytest.mark.parametrize("G", [4, 12])
@pytest.mark.parametrize("window, sinks", [(40, 3), (70, 33), (5, 0), (50, 64)])
def test_hidden_pages_and_tokens_may_hold_anything(G, window, sinks):
    """Pages that are left out replaced by one of NaNs, V scales and biases of hidden tokens (also behind a sequence's end)
    and exact K of hidden tail tokens set to NaN and infinities: the same bits."""
    D, H = 128, 2
    for bits in (4, 8):
        c, q = case(D, bits, G, H, torch.bfloat16, lens=[200, 77, 415, 90, 33], seed=5)
        want = run(c, q, D, bits, G, torch.bfloat16, window, sinks, splits=2)
        rec, body = c["records"], 2 * PAGE * (D if bits == 8 else D // 2)
        rec[0] = 255                                                     # block 0 is nobody's: fp16 NaNs all over
        meta = rec[..., body:].view(torch.float16)
        table = c["table"].cpu()
        for s, n in enumerate(c["lens"].tolist()):
            begin = max(0, n - window)
            for p in range(-(-n // PAGE)):
                hide = [t for t in range(PAGE) if sinks <= p * PAGE + t < begin or p * PAGE + t >= n]
                if len(hide) == PAGE and p * PAGE + PAGE <= begin:
                    c["table"][s, p] = 0
                else:
                    bad = torch.tensor([float("nan"), float("inf")] * PAGE, dtype=torch.float16, device=DEV)[:len(hide)]
                    meta[int(table[s, p]), :, 2 * D + torch.tensor(hide, dtype=torch.long)] = bad
                    meta[int(table[s, p]), :, 2 * D + PAGE + torch.tensor(hide, dtype=torch.long)] = -bad
            full = n // PAGE * PAGE
            for t in range(PAGE):
                if full + t >= n or sinks <= full + t < begin:
                    c["tail"][int(c["tidx"][s]), :, t] = float("nan") if t % 2 else float("inf")
        got = run(c, q, D, bits, G, torch.bfloat16, window, sinks, splits=2)
        assert bool(torch.isfinite(got).all()) and torch.equal(got, want)


@pytest.mark.parametrize("rot", [False, True])
@pytest.mark.parametrize("dtype, G", [(torch.bfloat16, 4), (torch.float16, 12), (torch.float32, 2)])
def test_append_under_a_window_is_the_two_calls(dtype, G, rot):
    """One launch of append_decode: the records, tails and outputs of append, then decode. The new token completes a page,
    starts one or lies inside; the window ends inside its page or far before it."""
    D, bits, H = 128, 4, 2
    lens = [1, 32, 33, 64, 70, 257, 320, 1000]
    for window, sinks, splits in ((1, 0, 1), (33, 2, 2), (200, 40, 3)):
        one, q = case(D, bits, G, H, dtype, lens, seed=6)
        two = {k: v.clone() for k, v in one.items()}
        g = torch.Generator().manual_seed(7)
        k, v = (torch.randn(len(lens), H, D, generator=g).to(dtype).to(DEV) for _ in range(2))
        got = run(one, q, D, bits, G, dtype, window, sinks, splits, rot=rot, k=k, v=v)
        kk.Ops(torch.device(DEV), D, bits, G, dtype).append(k, v, two["lens"], two["tidx"], two["records"], two["table"],
                                                            two["tail"], -1, False, rot=rot)
        want = run(two, q, D, bits, G, dtype, window, sinks, splits, rot=rot)
        for name in one:
            assert torch.equal(one[name], two[name]), name
        assert torch.equal(got, want)


def test_rotated_cache():
    """rot: q rotated (and rounded to its type) on load, the output rotated back: the reference does the same around the
    stored records."""
    D, bits, G, dtype = 128, 4, 4, torch.bfloat16
    c, q = case(D, bits, G, 2, dtype, seed=8)
    ops = kk.Ops(torch.device(DEV), D, bits, G, dtype)
    ref, most = decode_reference(ops.fwht(q), c, D, bits, G, D ** -0.5, 77, 9)
    H = torch.ones(1, 1, dtype=torch.float64)
    while H.shape[0] < D:
        H = torch.cat([torch.cat([H, H], 1), torch.cat([H, -H], 1)], 0)
    ref = ref @ (H / D ** 0.5)
    # the rotation adds D errors of 1 / sqrt(D) each: sqrt(D) times the bound of one, at most
    out = run(c, q, D, bits, G, dtype, 77, 9, splits=2, rot=True)
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= 2.5 * 2.0 ** -11 * most * D ** 0.5 + half_step(dtype) * (ref.abs() + 0.1)).all())


def test_a_window_over_everything_is_the_plain_decode():
    c, q = case(seed=9)
    ops = kk.Ops(torch.device(DEV), 128, 4, 4, torch.bfloat16)
    out = torch.empty_like(q)
    ops.decode(q, out, c["records"], c["table"], c["lens"], c["tidx"], c["tail"], 128 ** -0.5)
    ref, most = decode_reference(q, c, 128, 4, 4, 128 ** -0.5, 1025, 0)
    check(out, ref, most, torch.bfloat16)
    check(run(c, q, 128, 4, 4, torch.bfloat16, 1025, 0), ref, most, torch.bfloat16)


def test_replays_of_a_captured_step_follow_the_lengths():
    """A captured windowed step, replayed as the sequences grow in place: each replay is the eager call's bits."""
    D, bits, G, dtype = 128, 4, 4, torch.bfloat16
    c, q = case(D, bits, G, 2, dtype, lens=[900, 33, 500], seed=10)
    ops = kk.Ops(torch.device(DEV), D, bits, G, dtype, validate=False)
    splits = ops.splits(3, 2, 900 // PAGE, window=100, sinks=4)
    work = torch.empty(3 * 2 * splits * G * (D + 2), dtype=torch.float32, device=DEV)
    out, eager = torch.empty_like(q), torch.empty_like(q)

    def step(to):
        ops.decode(q, to, c["records"], c["table"], c["lens"], c["tidx"], c["tail"], D ** -0.5, splits, work, window=100, sinks=4)

    c["lens"].sub_(20)
    step(eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    for _ in range(4):
        c["lens"].add_(5)
        step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_on_another_stream():
    c, q = case(seed=11)
    want = run(c, q, 128, 4, 4, torch.bfloat16, 100, 4, splits=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(c, q, 128, 4, 4, torch.bfloat16, 100, 4, splits=2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_start_order_does_not_matter():
    D, G, dtype = 128, 4, torch.bfloat16
    c, q = case(seed=12)
    ops = kk.Ops(torch.device(DEV), D, 4, G, dtype)
    outs = []
    for order in (None, torch.arange(len(LENS) - 1, -1, -1, dtype=torch.int32, device=DEV)):
        out = torch.empty_like(q)
        ops.decode(q, out, c["records"], c["table"], c["lens"], c["tidx"], c["tail"], D ** -0.5, order=order, window=64, sinks=4)
        outs.append(out)
    assert torch.equal(*outs)


def test_refusals():
    c, q = case(seed=13)
    ops = kk.Ops(torch.device(DEV), 128, 4, 4, torch.bfloat16)
    args = (q, torch.empty_like(q), c["records"], c["table"], c["lens"], c["tidx"], c["tail"], 0.1)
    for kw in (dict(window=0), dict(window=-1), dict(window=2.0), dict(window=True), dict(window=4, sinks=-1), dict(sinks=3),
               dict(window=1 << 31), dict(window=8, n_splits=2)):
        with pytest.raises(ValueError):
            ops.decode(*args, **kw)
    with pytest.raises(ValueError):                                       # validated: a seen page outside the cache
        bad = dict(c, table=c["table"].clone())
        bad["table"][9, 0] = 10 ** 6
        run(bad, q, 128, 4, 4, torch.bfloat16, 40, 1)
    run(bad, q, 128, 4, 4, torch.bfloat16, 40, 0)                         # one that is not seen is not looked at
