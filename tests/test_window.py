"""Attention under a window on the CPU: the limit's checks, window_attention in fp32 products against 64 bits, with its
gradients, how the kernels' calls are planned, and what a cache or a model without the GPU refuses."""
from types import SimpleNamespace

import pytest
import torch

import kushkash_amd as kk
from _window_case import half_step, rows_reference, seen
from kushkash_amd import _attend, _window
from kushkash_amd._window import check_limit, pages_left_out


def rows(T, N, Hk, G, D, dtype, seed, batch=()):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*batch, n, h, D, generator=g).to(dtype) for n, h in ((T, Hk * G), (N, Hk), (N, Hk))]


def test_the_limit():
    assert check_limit(None, 0) == (0, 0) and check_limit(5, 0) == (5, 0) and check_limit(1 << 30, 1 << 30) == (1 << 30, 1 << 30)
    with pytest.raises(ValueError, match="sinks are for attention with a window"):
        check_limit(None, 4)
    for bad in (0, -1, 1.0, True, (1 << 30) + 1, "config"):
        with pytest.raises(ValueError, match="window must be an integer of 1"):
            check_limit(bad, 0)
    for bad in (-1, 2.0, False, (1 << 30) + 1):
        with pytest.raises(ValueError, match="sinks must be an integer of 0"):
            check_limit(7, bad)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 100])
@pytest.mark.parametrize("sinks", [0, 1, 32, 33, 64])
def test_pages_left_out_are_those_that_hold_nothing_seen(window, sinks):
    for p in range(0, 400, 7):
        pages = {j // 32 for j in seen(p, window, sinks)} | set(range(-(-sinks // 32)))      # the sinks' pages are kept
        first = (p - window + 1) // 32 if p >= window - 1 else 0
        assert pages_left_out(p, window, sinks) == len([x for x in range(first) if x not in pages])
    assert pages_left_out(10 ** 6, 0, 0) == 0


@pytest.mark.parametrize("T, N, window, sinks", [(1, 1, 1, 0), (1, 90, 7, 0), (5, 5, 2, 1), (64, 64, 16, 3), (33, 200, 40, 33),
                                                 (70, 70, 500, 0), (17, 130, 1, 200), (90, 91, 30, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_products(T, N, window, sinks, dtype):
    """fp32 products and softmax of N terms: each of the few roundings of a weight is 2^-24 of it, a score's D products of
    about 1 accumulate D / 2 steps at most, so a relative error of (D + N) 2^-24 of values of up to 5; then one rounding."""
    D, Hk, G = 24, 2, 3
    q, k, v = rows(T, N, Hk, G, D, dtype, T + N)
    out = kk.window_attention(q[None], k[None], v[None], window=window, sinks=sinks)[0]
    ref = rows_reference(q, k, v, D ** -0.5, window, sinks)
    most = float(v.double().abs().max())
    tol = (D * 8 + N) * 2.0 ** -24 * most + (half_step(dtype) * ref.abs() if dtype != torch.float32 else 0)
    assert out.dtype == dtype and bool(((out.double() - ref).abs() <= tol).all())


def test_products_in_blocks_of_queries_are_the_same(monkeypatch):
    q, k, v = rows(50, 120, 2, 2, 16, torch.float32, 3, batch=(2,))
    whole = _window._products(q, k, v, 33, 5, 0.25)
    parts = _window._products(q, k, v, 33, 5, 0.25, block_bytes=1)
    assert float((whole - parts).abs().max()) <= (16 * 8 + 120) * 2.0 ** -24 * 5


def test_ragged_rows_are_each_sequence_by_itself():
    spans = [(3, 9), (0, 0), (1, 40), (20, 20), (0, 5)]
    T, N = (sum(s[i] for s in spans) for i in (0, 1))
    q, k, v = rows(T, N, 2, 2, 16, torch.float32, 4)
    out = torch.full_like(q, 7.0)
    got = kk.window_attention(q, k, v, window=6, sinks=2, spans=spans, out=out)
    assert got is out
    a = c = 0
    for t, n in spans:
        if t:
            one = kk.window_attention(q[None, a:a + t], k[None, c:c + n], v[None, c:c + n], window=6, sinks=2)[0]
            assert torch.equal(got[a:a + t], one)
        a, c = a + t, c + n


def test_a_window_over_everything_is_causal_attention():
    q, k, v = rows(12, 12, 1, 2, 8, torch.float64, 5, batch=(1,))
    got = kk.window_attention(q.float(), k.float(), v.float(), window=100)
    want = torch.nn.functional.scaled_dot_product_attention(*(x.transpose(1, 2).repeat_interleave(r, 1)
                                                              for x, r in ((q, 1), (k, 2), (v, 2))), is_causal=True)
    assert float((got.double() - want.transpose(1, 2)).abs().max()) <= (8 * 8 + 12) * 2.0 ** -24 * 5


def formula_gradients(q, k, v, do, scale, window, sinks):
    """dq, dk, dv in 64 bits by the softmax's derivative: ds = p (do.v - sum p do.v)."""
    q, k, v, do = (x.double() for x in (q, k, v, do))
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    N = k.shape[0]
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(T):
        js = seen(N - T + t, window, sinks)
        for h in range(Hq):
            K, V = k[js, h // G], v[js, h // G]
            p = torch.softmax(scale * K @ q[t, h], 0)
            dp = V @ do[t, h]
            ds = p * (dp - (p * dp).sum()) * scale
            dq[t, h] = ds @ K
            dk[js, h // G] += ds[:, None] * q[t, h]
            dv[js, h // G] += p[:, None] * do[t, h]
    return dq, dk, dv


@pytest.mark.parametrize("T, N, window, sinks", [(1, 1, 1, 0), (9, 9, 3, 1), (7, 30, 5, 2), (6, 20, 40, 0)])
def test_gradients(T, N, window, sinks):
    """Of shared kv heads, in fp32 against the formula: about 4 (D + N) roundings of 2^-24 in each of up to T G terms of a sum;
    and the formula against central differences in 64 bits."""
    D, Hk, G = 8, 2, 3
    q, k, v = rows(T, N, Hk, G, D, torch.float32, 11)
    do = rows(T, N, Hk, G, D, torch.float32, 12)[0]
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    kk.window_attention(*(x[None] for x in leaves), window=window, sinks=sinks)[0].backward(do)
    want = formula_gradients(q, k, v, do, D ** -0.5, window, sinks)
    for x, w in zip(leaves, want):
        tol = 4 * (D + N) * 2.0 ** -24 * (T * G) ** 0.5 * max(1.0, float(w.abs().max())) * 4
        assert float((x.grad.double() - w).abs().max()) <= tol
    inputs = [x.double() for x in (q, k, v)]
    for which, w in enumerate(want):                        # along the gradient: |w|^2
        if not float(w.norm()):
            continue
        e = 1e-5 / float(w.norm())
        value = []
        for s in (e, -e):
            moved = [x + s * w if i == which else x for i, x in enumerate(inputs)]
            value.append(float((rows_reference(*moved, D ** -0.5, window, sinks) * do.double()).sum()))
        assert abs((value[0] - value[1]) / (2 * e) - float(w.norm()) ** 2) <= 1e-6 * max(1.0, float(w.norm()) ** 2)


def test_rows_hidden_from_every_query_may_hold_anything():
    q, k, v = rows(4, 60, 1, 2, 8, torch.float32, 6, batch=(1,))
    want = kk.window_attention(q, k, v, window=5, sinks=2)
    k[:, 2:52] = float("nan")
    k[:, 30] = float("inf")
    v[:, 2:52] = float("nan")
    assert torch.equal(kk.window_attention(q, k, v, window=5, sinks=2), want)


def test_refusals_of_window_attention():
    q, k, v = rows(4, 6, 2, 2, 8, torch.float32, 7, batch=(1,))
    call = kk.window_attention
    for bad, match in [
        (lambda: call(q, k, v, window=None), "needs a window"),
        (lambda: call(q, k, v, window=0), "window must be an integer"),
        (lambda: call(q, k, v, window=3, sinks=-1), "sinks must be"),
        (lambda: call(q[0], k, v, window=3), "must be .rows, heads, dim. with spans"),
        (lambda: call(q, k, v, window=3, spans=[(4, 6)]), "must be .rows, heads, dim. with spans"),
        (lambda: call(q, k, v, window=3, cu=(q, q)), "cu needs spans"),
        (lambda: call(q, k, v[:, 1:], window=3), "one shape"),
        (lambda: call(q[:, :, :3], k, v, window=3), "multiple of their heads"),
        (lambda: call(q[..., :4], k, v, window=3), "head_dim"),
        (lambda: call(q.double(), k, v, window=3), "one floating-point dtype"),
        (lambda: call(q.int(), k.int(), v.int(), window=3), "one floating-point dtype"),
        (lambda: call(q, k, v, window=3, scale=0.0), "scale must be positive"),
        (lambda: call(q, k, v, window=3, scale=float("nan")), "scale must be positive"),
        (lambda: call(q, k[:, :3], v[:, :3], window=3), "as many rows or more"),
        (lambda: call(q, k.repeat(2, 1, 1, 1), v.repeat(2, 1, 1, 1), window=3), "q's batch"),
        (lambda: call(q, k, v, window=3, out=q[:, :2]), "out must have q's shape"),
        (lambda: call(q[0], k[0], v[0], window=3, spans=[(4, 3)]), "as many keys as queries"),
        (lambda: call(q[0], k[0], v[0], window=3, spans=[(-1, 3), (5, 3)]), "as many keys as queries"),
        (lambda: call(q[0], k[0], v[0], window=3, spans=[(3, 6)]), "spans hold 3 queries"),
        (lambda: call(q[0], k[0], v[0], window=3, spans=[(4, 6)], cu=(torch.zeros(2), torch.zeros(2))), "int32"),
    ]:
        with pytest.raises(ValueError, match=match):
            bad()
    assert call(q[:, :0], k, v, window=3).shape == (1, 0, 4, 8)


# ------------------------------------------------------------------ plans
@pytest.mark.parametrize("group", [1, 4, 7])
@pytest.mark.parametrize("window, sinks", [(1, 0), (64, 0), (65, 1), (100, 64), (1000, 65)])
def test_no_row_tile_sees_more_key_tiles_than_planned(group, window, sinks):
    """window_tiles bounds the key tiles (64 keys) that hold a seen key of any tile of 128 query rows, wherever it lies."""
    bound = _attend.window_tiles(window, sinks, 128, group)
    tokens = -(-128 // group) + 1                            # that a tile's rows can belong to
    for p in (0, 63, 64, 500, 4095, 4096, 5001):
        for part in (tokens, tokens - 1):
            tiles = {j // 64 for t in range(p, p + part) for j in seen(t, window, sinks)}
            assert len(tiles) <= bound, (p, part)


def test_row_tiles():
    assert _attend.row_tiles([(0, 5), (1, 9), (32, 32), (33, 40)], 4, 4) == 0 + 1 + 1 + 2
    assert _attend.row_tiles([(100, 100, 3)], 2, 8) == 3


@pytest.mark.parametrize("D", [64, 128, 256])
def test_plans_split_only_into_parts_that_hold_tiles_and_fit_the_scratch(D):
    for T in (1, 20, 150, 700, 4096):
        for N in (T, T + 90, T + 3000):
            for window in (1, 64, 700, 2048):
                for hkv, group in ((1, 1), (2, 8), (8, 4)):
                    waves, chunk = _attend.plan([(T, N, 2)], group, hkv, D, 2 * T, True, 1 << 28, window, 5)
                    tiles = min(-(-N // 64), _attend.window_tiles(window, 5, 32 * waves, group))
                    assert waves in (4, 8) and (chunk == 0 or (chunk >= 3 and chunk < tiles))
                    if chunk:
                        assert -(-tiles // chunk) * 2 * T * hkv * group * (D + 2) * 4 <= _attend.PARTIAL_BYTES


def test_what_the_native_plan_leaves_to_the_checks():
    """Shapes that the kernel does not take, or that see every key: None, so that the checks of the call answer."""
    plan = _attend._window_plan
    assert plan((1, 9, 4, 64), (1, 50, 2, 64), None, 1 << 28, 7, 0)[:3] == (9, 50, 4)
    for q, k, spans, window in [
        ((1, 9, 4, 80), (1, 50, 2, 80), None, 7), ((1, 9, 3, 64), (1, 50, 2, 64), None, 7), ((1, 9, 4, 64), (2, 50, 2, 64), None, 7),
        ((1, 0, 4, 64), (1, 50, 2, 64), None, 7), ((1, 60, 4, 64), (1, 50, 2, 64), None, 7), ((1, 9, 4, 64), (1, 50, 2, 64), None, 50),
        ((9, 4, 64), (50, 2, 64), ((9, 49),), 7), ((9, 4, 64), (50, 2, 64), ((8, 50),), 7), ((9, 4, 64), (50, 2, 64), ((9, 8), (0, 42)), 7),
        ((9, 4, 64), (50, 2, 64), None, 7), ((1, 9, 4, 64), (50, 2, 64), None, 7),
    ]:
        assert plan(q, k, spans, 1 << 28, window, 0) is None, (q, k, spans)


# ------------------------------------------------------------------ caches and models
def test_a_window_is_for_the_gpu_kernels():
    with pytest.raises(ValueError, match="a window is for the GPU kernels"):
        kk.KushCache(2, 2, 4, 64, device="cpu", window=64)
    with pytest.raises(ValueError, match="a window is for the GPU kernels"):
        kk.KushCache(2, 2, 4, 64, device="cpu", window=[None, 64], sinks=4)
    with pytest.raises(ValueError, match="one per layer"):
        kk.KushCache(2, 2, 4, 64, device="cpu", window=[64])
    with pytest.raises(ValueError, match="sinks are for attention with a window"):
        kk.KushCache(2, 2, 4, 64, device="cpu", sinks=4)
    with pytest.raises(ValueError, match="window must be an integer"):
        kk.KushCache(2, 2, 4, 64, device="cpu", window=0)
    cache = kk.KushCache(2, 2, 4, 64, device="cpu", window=[None, None])
    assert cache.layer_limit(0) == (0, 0)


def test_splits_count_the_pages_that_are_seen():
    ops = SimpleNamespace(gpu=True, sms=256, D=128, bits=4, G=4)
    full = kk.Ops.splits
    plain = full(ops, 1, 8, 4096)
    assert full(ops, 1, 8, 4096, window=64) <= plain
    assert full(ops, 1, 8, 4096, window=1 << 20) == plain


def test_layer_windows():
    from kushkash_amd.hf import _check_config, layer_windows
    cfg = lambda **kw: SimpleNamespace(num_hidden_layers=3, **kw)  # noqa: E731
    assert layer_windows(cfg(sliding_window=None)) == [None] * 3
    assert layer_windows(cfg(sliding_window=64, max_position_embeddings=100)) == [64] * 3
    assert layer_windows(cfg(sliding_window=200, max_position_embeddings=100)) == [None] * 3
    kinds = ["sliding_attention", "full_attention", "sliding_attention"]
    assert layer_windows(cfg(sliding_window=64, layer_types=kinds)) == [64, None, 64]
    assert layer_windows(cfg(sliding_window=64, layer_types=["full_attention"] * 3)) == [None] * 3
    for bad in (cfg(sliding_window=64, layer_types=["chunked_attention"] * 3), cfg(sliding_window=64, layer_types=kinds[:2]),
                cfg(use_sliding_window=True), cfg(sliding_window=None, layer_types=kinds)):
        with pytest.raises(NotImplementedError, match="kushkash"):
            _check_config(bad, sliding_window=True)
    _check_config(cfg(sliding_window=64, layer_types=kinds), sliding_window=True)
    with pytest.raises(NotImplementedError, match="softcapping"):
        _check_config(cfg(sliding_window=64, layer_types=kinds, attn_logit_softcapping=30.0), sliding_window=True)
    with pytest.raises(NotImplementedError, match="sliding-window"):
        _check_config(cfg(sliding_window=64, layer_types=kinds))


def test_windows_of_a_model_s_cache():
    transformers = pytest.importorskip("transformers")
    cfg = transformers.MistralConfig(num_hidden_layers=2, sliding_window=48, max_position_embeddings=512)
    assert kk.KushHFCache(cfg).windows == [None, None]
    assert kk.KushHFCache(cfg, window="config").windows == [48, 48]
    assert kk.KushHFCache(cfg, window=9, sinks=2).windows == [9, 9]
    with pytest.raises(ValueError, match="'config'"):
        kk.KushHFCache(cfg, window="sliding")


@pytest.mark.parametrize("extra, match", [(dict(s_aux=torch.zeros(4)), "learned sink logits"), (dict(softcap=30.0), "softcapping")])
def test_attention_with_more_than_a_window_is_refused(extra, match):
    from kushkash_amd import hf
    key = torch.zeros(1, 2, 1, 64)
    setattr(key, hf._ROUTE, (SimpleNamespace(kv=object()), 0))
    with pytest.raises(NotImplementedError, match=match):
        hf.kush_attention(None, torch.zeros(1, 4, 1, 64), key, key, None, **extra)


def test_a_sliding_layer_needs_its_window_in_the_cache():
    from kushkash_amd import hf
    cfg = SimpleNamespace(sliding_window=64, max_position_embeddings=512)
    for limit in ((0, 0), (65, 0)):
        key = torch.zeros(1, 2, 1, 64)
        setattr(key, hf._ROUTE, (SimpleNamespace(kv=SimpleNamespace(layer_limit=lambda layer: limit)), 0))
        with pytest.raises(RuntimeError, match="window='config'"):
            hf.kush_attention(SimpleNamespace(config=cfg), torch.zeros(1, 4, 1, 64), key, key, None, sliding_window=64)


def test_generate_refuses_before_anything_runs():
    ids = torch.zeros(1, 3, dtype=torch.long)
    for kw, match in [(dict(cache=object(), window=5), "window and sinks are the cache's"),
                      (dict(cache=object(), sinks=5), "window and sinks are the cache's"),
                      (dict(top_p=-0.1), "must be >= 0"), (dict(min_p=float("nan")), "must be >= 0")]:
        with pytest.raises(ValueError, match=match):
            kk.generate(None, ids, 4, **kw)
