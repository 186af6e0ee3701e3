"""block_table and step_maps on the GPU, entry by entry against their definition; a windowed serving step put together."""
import random

import pytest
import torch

import kushkash_amd as kk
from _maps_case import check
from _window_case import PAGE, half_step, seen

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (32, 1), (33, 32), (100, 33), (500, 4), (1 << 30, 0)])
def test_maps(window, sinks):
    check(kk, torch, [1], [0], DEV, window, sinks)
    check(kk, torch, [0], [0], DEV, window, sinks)
    check(kk, torch, [0, 5, 0, 32, 33, 1, 1, 700], [40, 0, 0, 31, 32, 63, 64, 999], DEV, window, sinks)
    check(kk, torch, [], [], DEV, window, sinks)
    rng = random.Random(window)
    for n in (3, 64, 300):
        check(kk, torch, [rng.randint(0, 80) for _ in range(n)], [rng.choice([0, rng.randint(1, 3000)]) for _ in range(n)], DEV,
              window, sinks, seed=n)


def test_one_long_request():
    check(kk, torch, [9001], [40007], DEV)
    check(kk, torch, [9001, 1], [40007, 3], DEV, 4096, 100)


def test_lengths_past_the_sizes_and_the_table_stay_inside():
    """Device lengths that need more than the sizes, or more pages than the table has: cut off, what lies behind the arrays
    untouched."""
    sizes = kk.map_sizes([4, 4], [40, 40])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.arange(1, 5, dtype=torch.int32, device=DEV).view(2, 2)
    for new, history in (([4, 5000], [40, 40]), ([4, 4], [40, 90000]), ([-7, 4], [40, -3]), ([2, 1], [3, 4])):
        m = kk.step_maps(i32(new), i32(history), i32([1, 0]), table, sizes)
        torch.cuda.synchronize()
        assert m.job_seq.numel() == 2 and m.slot_map.numel() == 8 and bool((m.tail_blk >= 0).all())
        assert bool((m.slot_map[:1] >= 0).all())


@pytest.mark.parametrize("wide_req", [torch.int32, torch.int64])
@pytest.mark.parametrize("wide_lens", [torch.int32, torch.int64])
def test_block_table(wide_req, wide_lens):
    g = torch.Generator().manual_seed(0)
    rows, cols = 11, 1000
    tokens = torch.randint(0, 1 << 30, (rows, cols), generator=g, dtype=torch.int32)
    lens = [0, 1, 31, 32, 33, 1000, 999, 500]
    req = torch.randperm(rows, generator=g)[:len(lens)]
    for pages in (0, 1, 32, 40, 300):
        want = torch.zeros(len(lens), pages, dtype=torch.int32)
        for r, n in enumerate(lens):
            for p in range(min(pages, -(-n // PAGE))):
                want[r, p] = tokens[req[r], p * PAGE] // PAGE
        buf = torch.full((len(lens) + 1, pages + 5), -9, dtype=torch.int32, device=DEV)
        out = (buf[:len(lens), :pages], *(torch.full((len(lens),), -9, dtype=torch.int32, device=DEV) for _ in range(2)))
        args = (tokens.to(DEV), req.to(wide_req).to(DEV), torch.tensor(lens, dtype=wide_lens, device=DEV), pages)
        for got in (kk.block_table(*args), kk.block_table(*args, out=out)):
            assert torch.equal(got[0].cpu(), want) and got[1].tolist() == lens and got[2].tolist() == req.tolist()
            assert all(x.dtype == torch.int32 for x in got)
        assert bool((buf[-1] == -9).all()) and bool((buf[:, pages:] == -9).all())      # rows and columns behind: as they were


def test_block_table_of_requests_and_lengths_outside_the_map():
    tokens = torch.arange(64, dtype=torch.int32, device=DEV).view(1, 64) * 32
    req = torch.tensor([0, 1, -1], device=DEV)
    got = kk.block_table(tokens, req, torch.tensor([500, 64, 64], device=DEV), 4)
    assert got[0].tolist() == [[0, 32, 0, 0], [0, 0, 0, 0], [0, 0, 0, 0]] and got[1].tolist() == [500, 64, 64]


def test_a_captured_table_follows_the_lengths():
    tokens = torch.randint(0, 1 << 20, (6, 640), dtype=torch.int32, device=DEV)
    req, lens = torch.arange(5, device=DEV), torch.tensor([1, 31, 64, 100, 600], device=DEV)
    out = kk.block_table(tokens, req, lens, 20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kk.block_table(tokens, req, lens, 20, out=out)
    for _ in range(3):
        lens.add_(13)
        req.copy_((req + 1) % 6)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, kk.block_table(tokens, req, lens, 20)))


@pytest.mark.parametrize("bits, rot", [(4, False), (8, False), (4, True)])
def test_a_windowed_serving_session(bits, rot):
    """The operators together, as a server runs them: prompts of ragged lengths, a second turn over the history that the
    window leaves, then decode steps whose tables come from the token map, and a token drawn from their outputs. The
    attention of every step is compared with the definition over the rows as they were given: K and V go through records
    of `bits` bits, so the comparison is to the quantization's own error (relative 2-norm: an int4 page's codes are 1 / 15
    of its range apart, uniform over half a step of it, int8's 1 / 255; a normal page's range is about 4 sigma: 8 % and
    0.5 % of K and V; weights of a score off by 8 % of |q| ~ 8 % once more, together below 0.2 and 0.02)."""
    D, H, G, dtype, window, sinks = 128, 2, 4, torch.bfloat16, 70, 5
    g = torch.Generator().manual_seed(bits)
    ops = kk.Ops(torch.device(DEV), D, bits, G, dtype)
    R, context = 3, 640
    cache = torch.zeros(200, H, kk.record_bytes(D, bits), dtype=torch.uint8, device=DEV)
    tails = torch.zeros(8, H, PAGE, D, dtype=dtype, device=DEV)
    blocks = torch.randperm(200, generator=g)[:8 * context // PAGE].view(8, -1)
    token_map = (blocks[:, :, None] * PAGE + torch.arange(PAGE)).view(8, -1).to(torch.int32).to(DEV)
    req = torch.tensor([6, 1, 3], device=DEV)
    rows = [[torch.zeros(0, H, D), torch.zeros(0, H, D)] for _ in range(R)]           # K, V as given
    lens = [0] * R
    worst = 0.0

    def reference(r, q, first):
        K, V = rows[r]
        out = torch.empty(q.shape, dtype=torch.float64)
        for t in range(q.shape[0]):
            js = seen(first + t, window, sinks)
            for i in range(H * G):
                s = q[t, i].double() @ K[js, i // G].double().T * D ** -0.5
                out[t, i] = torch.softmax(s, -1) @ V[js, i // G].double()
        return out

    def compare(got, want):
        nonlocal worst
        worst = max(worst, float((got.double().cpu() - want).norm() / want.norm()))

    def rand(n, h):
        return torch.randn(n, h, D, generator=g).to(dtype)

    for new in ([45, 64, 200], [30, 7, 33]):                                          # two prefill steps
        T = torch.tensor(new, dtype=torch.int32, device=DEV)
        old = torch.tensor(lens, dtype=torch.int32, device=DEV)
        table, _, slots = kk.block_table(token_map, req, (old + T), context // PAGE)
        m = kk.step_maps(T, old, slots, table, kk.map_sizes(new, lens, window=window, sinks=sinks))
        q, k, v = (rand(sum(new), h) for h in (H * G, H, H))
        kd, vd = k.to(DEV), v.to(DEV)
        kp, vp = (torch.empty(m.sizes.keys, H, D, dtype=dtype, device=DEV) for _ in range(2))
        ops.unpack(cache, m.page_blk, m.page_dst, m.tail_blk, m.tail_info.view(-1), tails, kd, vd, m.new_dst, kp, vp, rot)
        spans = list(zip(new, (m.key_start[1:] - m.key_start[:-1]).tolist()))
        out = kk.window_attention(q.to(DEV), kp, vp, window=window, sinks=sinks, spans=spans, cu=(m.q_start, m.key_start))
        ops.write(kd, vd, m.q_start, m.seq_lens, slots, m.job_seq, m.job_page, cache, table, tails, fused=True, rot=rot)
        a = 0
        for r, t in enumerate(new):
            rows[r] = [torch.cat([x, y[a:a + t].float()]) for x, y in zip(rows[r], (k, v))]
            compare(out[a:a + t], reference(r, q[a:a + t], lens[r]))
            lens[r] += t
            a += t
        assert m.seq_lens.tolist() == lens
    seq = torch.tensor(lens, device=DEV)
    weight = torch.randn(H * G * D, 1000, generator=g).to(DEV) / 8
    for step in range(40):                                                            # decode steps over page borders
        seq += 1
        table, sl, slots = kk.block_table(token_map, req, seq, context // PAGE)
        q, k, v = (rand(R, h) for h in (H * G, H, H))
        out = torch.empty(R, H * G, D, dtype=dtype, device=DEV)
        splits = ops.splits(R, H, context // PAGE, window=window, sinks=sinks)
        work = torch.empty(R * H * splits * G * (D + 2), dtype=torch.float32, device=DEV)
        ops.append_decode(k.to(DEV), v.to(DEV), q.to(DEV), out, cache, table, sl, slots, tails, D ** -0.5, splits, work, rot=rot,
                          window=window, sinks=sinks)
        for r in range(R):
            rows[r] = [torch.cat([x, y[r:r + 1].float()]) for x, y in zip(rows[r], (k, v))]
            if step % 7 == 0:
                compare(out[r:r + 1], reference(r, q[r:r + 1], lens[r]))
            lens[r] += 1
        tokens = kk.sample(out.view(R, -1).float() @ weight, torch.rand(R, device=DEV), temperature=0.8, top_k=20, top_p=0.9)
        assert bool(((tokens >= 0) & (tokens < 1000)).all())
    assert worst < (0.2 if bits == 4 else 0.02), worst


@pytest.mark.parametrize("krot", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kush_cache_under_a_window(dtype, krot):
    """KushCache(window=, sinks=), a layer with and one without: a prompt chunk by chunk, then tokens one by one, against
    window_attention's products over the cache's own dequantized rows (and, for a chunk, its rows as given)."""
    B, H, G, D, window, sinks = 2, 2, 4, 64, 50, 3
    cache = kk.KushCache(2, H, H * G, D, batch_size=B, bits=8, device=DEV, dtype=dtype, window=[window, None], sinks=sinks,
                         rotate=krot, rotate_in_kernels=krot)
    g = torch.Generator().manual_seed(1)
    tol = dict(rtol=0, atol=20 * half_step(dtype) if dtype == torch.bfloat16 else 4e-3)   # bf16: a few roundings of values ~ 1

    def rand(h, t):
        return torch.randn(B, h, t, D, generator=g).to(dtype).to(DEV)

    def want(layer, q, k, v):
        K, V = (torch.cat([x, y], 2) for x, y in zip(cache.dequantize(layer) if cache.length(layer) else (k[:, :, :0], v[:, :, :0]), (k, v)))
        w, s = (window, sinks) if layer == 0 else (1 << 20, 0)
        x = [t.float().transpose(1, 2) for t in (q, K, V)]
        return kk.window_attention(*x, window=w, sinks=s).transpose(1, 2)

    for T in (33, 100, 7):
        for layer in (0, 1):
            q, k, v = rand(H * G, T), rand(H, T), rand(H, T)
            ref = want(layer, q, k, v)
            torch.testing.assert_close(cache.attend_chunk(layer, q, k, v).float(), ref, **tol)
            cache.write(layer, k, v)
    for step in range(20):
        if step == 3:
            cache.freeze(200)
        for layer in (0, 1):
            q, k, v = rand(H * G, 1), rand(H, 1), rand(H, 1)
            ref = want(layer, q, k, v)
            out = cache.append_attend(layer, q[:, :, 0], k, v)
            if (cache.length(layer)) % PAGE:                              # (a completed page's new keys are quantized by now)
                torch.testing.assert_close(out.float(), ref[:, :, 0], **tol)


def test_refusals():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    sizes = kk.map_sizes([1, 2], [3, 4])
    ok = [i32([1, 2]), i32([3, 4]), i32([0, 1]), torch.zeros(2, 4, dtype=torch.int32, device=DEV)]
    kk.step_maps(*ok, sizes)
    for i, bad in ((0, i32([1])), (0, ok[0].long()), (1, ok[1].cpu()), (2, i32([[0, 1]])), (3, ok[3][:1]), (3, ok[3].long()),
                   (3, torch.zeros(4, 2, dtype=torch.int32, device=DEV).t())):
        with pytest.raises(ValueError):
            kk.step_maps(*(bad if j == i else x for j, x in enumerate(ok)), sizes)
    tokens, req, lens = torch.zeros(2, 64, dtype=torch.int32, device=DEV), torch.tensor([0], device=DEV), torch.tensor([5], device=DEV)
    for args in ((tokens.long(), req, lens, 2), (tokens, req.float(), lens, 2), (tokens, req, lens.cpu(), 2), (tokens, req, lens, -1),
                 (tokens, req, torch.tensor([5, 6], device=DEV), 2), (tokens.t(), req, lens, 2)):
        with pytest.raises(ValueError):
            kk.block_table(*args)
    good = kk.block_table(tokens, req, lens, 2)
    with pytest.raises(ValueError):
        kk.block_table(tokens, req, lens, 3, out=good)


@pytest.mark.parametrize("new, history", [([2 ** 31 - 1, 2 ** 31 - 1, 4], [2 ** 31 - 1, 2 ** 31 - 1, 40]), ([1] * 300, [2 ** 31 - 1] * 300),
                                          ([2 ** 31 - 32] * 70, [31] * 70), ([4, 4, 4], [2 ** 31 - 1, 0, 2 ** 30])])
@pytest.mark.parametrize("window", [0, 100])
def test_sums_of_lengths_that_pass_32_bits_stay_inside(new, history, window):
    """Lengths that no cache has (a buffer not yet filled): nothing before or behind the arrays is written."""
    from kushkash_amd import _lib
    n, jobs, pages, tails, tokens, guard = len(new), 5, 6, 3, 7, 64
    counts = [n + 1, n + 1, n, jobs, jobs, pages, pages, tails, 3 * tails, tokens, 2 * tokens]
    buf = torch.full((sum(counts) + guard * (len(counts) + 1) + len(counts),), -99, dtype=torch.int32, device=DEV)
    at, spots, mine = guard, [], torch.zeros(buf.numel(), dtype=torch.bool)
    for c in counts:
        at += at & 1                                                      # (the int64 array 8-byte aligned)
        spots.append(buf.data_ptr() + 4 * at)
        mine[at:at + c] = True
        at += c + guard
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    lens, table = (i32(new), i32(history), i32(list(range(n)))), torch.ones(n, 4, dtype=torch.int32, device=DEV)
    _lib.call("kush_step_maps", *(x.data_ptr() for x in lens), table.data_ptr(), 4, 4, n, window, 0, jobs, pages, tails, tokens, *spots,
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert bool((buf.cpu()[~mine] == -99).all())
