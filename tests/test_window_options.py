"""The limits that a model's cache takes: refused where it is built, as KushCache and Ops refuse them."""
import pytest

import kushkash_amd as kk

transformers = pytest.importorskip("transformers")


def config(window):
    return transformers.MistralConfig(num_hidden_layers=2, sliding_window=window, max_position_embeddings=512)


@pytest.mark.parametrize("kw, match", [
    (dict(sinks=4), "sinks are for attention with a window"), (dict(window=None, sinks=1), "sinks are for"),
    (dict(window=0), "window must be"), (dict(window=-3), "window must be"), (dict(window=2.5), "window must be"),
    (dict(window=True), "window must be"), (dict(window=(1 << 30) + 1), "window must be"), (dict(window=64, sinks=-1), "sinks must be"),
    (dict(window=64, sinks=1.5), "sinks must be"), (dict(window="config", sinks=-1), "sinks must be"), (dict(window="all"), "'config'"),
])
@pytest.mark.parametrize("sliding", [48, None])
def test_limits_that_no_cache_has(kw, match, sliding):
    with pytest.raises(ValueError, match=match):
        kk.KushHFCache(config(sliding), **kw)


def test_limits_that_a_cache_has():
    assert kk.KushHFCache(config(48), window=64, sinks=4).windows == [64, 64]
    assert kk.KushHFCache(config(48)).windows == [None, None]
    cache = kk.KushHFCache(config(48), window="config", sinks=4)
    assert cache.windows == [48, 48] and cache.sinks == 4
    assert kk.KushHFCache(config(None), window="config", sinks=4).windows == [None, None]
