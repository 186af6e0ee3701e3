"""Windows, top-p and random numbers through the Hugging Face entry points, on the GPU kernels: a sliding-window model
against its own sdpa attention, a window given to a full-attention model, and generate's sampling.

References run in fp32, as in the tests of the entry points without a window."""
import copy

import pytest
import torch

import kushkash_amd as kk

pytestmark = pytest.mark.gpu
transformers = pytest.importorskip("transformers")
DEV = "cuda"
COMMON = dict(vocab_size=256, hidden_size=256, intermediate_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=64,
              max_position_embeddings=4096)


def sliding(window=40, layers=2, dtype=torch.float32):
    from transformers import MistralConfig, MistralForCausalLM
    torch.manual_seed(0)
    return MistralForCausalLM(MistralConfig(**COMMON, num_hidden_layers=layers, sliding_window=window)).to(DEV, dtype).eval()


def full(layers=2, dtype=torch.float32):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    return LlamaForCausalLM(LlamaConfig(**COMMON, num_hidden_layers=layers)).to(DEV, dtype).eval()


def prompt(n, rows=2, seed=1):
    return torch.randint(0, 256, (rows, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


@torch.no_grad()
def test_a_sliding_window_model():
    """The prompt's logits are those of the model's own attention (fp32: 1e-4 as without a window), 40 int8 decode steps
    stay within 5 % of its largest logit, and full attention over the same tokens does not."""
    from transformers import DynamicCache
    model = sliding()
    ref = copy.deepcopy(model)
    ref.set_attn_implementation("sdpa")
    whole = copy.deepcopy(ref)
    whole.config.sliding_window = None
    kk.enable(model, sliding_window=True)
    cache, rc = kk.KushHFCache(model.config, bits=8, window="config"), DynamicCache()
    ids = prompt(130)
    out, want = model(ids, past_key_values=cache, use_cache=True).logits, ref(ids, past_key_values=rc, use_cache=True).logits
    assert float((out - want).abs().max()) < 1e-4
    assert float((whole(ids).logits - want).abs().max()) > 1e-2            # the window matters
    assert cache.kv.layer_limit(1) == (40, 0)
    seen = ids
    for _ in range(40):
        nxt = out[:, -1:].argmax(-1)
        seen = torch.cat([seen, nxt], 1)
        out = model(nxt, past_key_values=cache, use_cache=True).logits
        want = ref(seen, use_cache=False).logits[:, -1:]
        assert float((out - want).abs().max()) < 0.05 * float(want.abs().max())


@torch.no_grad()
def test_a_sliding_window_model_needs_its_windows():
    model = sliding()
    with pytest.raises(NotImplementedError, match="sliding-window"):
        kk.enable(model)
    with pytest.raises(NotImplementedError, match="sliding-window"):
        kk.generate(model, prompt(20), 2)
    kk.enable(model, sliding_window=True)
    for kw in ({}, dict(window=41)):
        with pytest.raises(RuntimeError, match="window='config'"):
            model(prompt(20), past_key_values=kk.KushHFCache(model.config, **kw), use_cache=True)
    model(prompt(20), past_key_values=kk.KushHFCache(model.config, window=30), use_cache=True)       # a smaller one will do
    given = sliding()
    cache = kk.KushHFCache(given.config, window="config")
    kk.generate(given, prompt(70), 3, cache=cache)                                                   # enabled for that cache
    assert cache.get_seq_length() == 72


@torch.no_grad()
@pytest.mark.parametrize("bits, rotate, dtype", [(4, True, torch.float16), (8, False, torch.bfloat16)])
@pytest.mark.parametrize("chunk", [1024, 48])
def test_tokens_outside_the_window_do_not_matter(bits, rotate, dtype, chunk):
    """One layer: a step's logits are bit for bit the same when tokens change in pages between the sinks' and the window's,
    with the prompt in one piece and in chunks, and other logits follow from a change inside."""
    model = full(layers=1, dtype=dtype)
    kk.enable(model)
    ids = prompt(200)
    logits = []
    for at in (None, range(32, 128), [150]):
        x = ids.clone()
        if at is not None:
            x[:, list(at)] = (x[:, list(at)] + 7) % 256
        cache = kk.KushHFCache(model.config, bits=bits, rotate=rotate, window=64, sinks=5, max_length=400)
        for c in range(0, 200, chunk):
            last = model(x[:, c:c + chunk], past_key_values=cache, use_cache=True).logits[:, -1]
        step = model(ids[:, :1], past_key_values=cache, use_cache=True).logits[:, -1]
        logits.append((last, step))
    for i in (0, 1):
        assert bool(torch.isfinite(logits[0][i]).all())
        assert torch.equal(logits[0][i], logits[1][i])
        assert not torch.equal(logits[0][i], logits[2][i])


@torch.no_grad()
def test_a_window_over_everything_generates_the_same_tokens():
    model = full()
    ids = prompt(90)
    want = kk.generate(model, ids, 40, bits=8)
    assert torch.equal(kk.generate(model, ids, 40, bits=8, window=1000, sinks=4), want)


@torch.no_grad()
@pytest.mark.parametrize("graph", [True, False])
def test_generate_under_a_window(graph):
    """Greedy tokens, eager and replayed, are those of a loop over the model's forward with such a cache."""
    model = full()
    ids = prompt(150)
    got = kk.generate(model, ids, 60, window=70, sinks=4, cuda_graph=graph)
    cache = kk.KushHFCache(model.config, window=70, sinks=4, max_length=210)
    out, want = model(ids, past_key_values=cache, use_cache=True).logits, ids
    for _ in range(60):
        tok = out[:, -1:].argmax(-1)
        want = torch.cat([want, tok], 1)
        out = model(tok, past_key_values=cache, use_cache=True).logits
    assert got.shape == want.shape
    same = (got == want).float().mean()
    assert float(same) > 0.9, same                                         # equal but for near ties: split counts differ


@torch.no_grad()
def test_generate_samples_from_given_random_numbers():
    model = full()
    ids = prompt(40)

    def run(seed=3, **kw):
        return kk.generate(model, ids, 24, do_sample=True, generator=torch.Generator(DEV).manual_seed(seed), cuda_graph=False,
                           **kw)

    assert torch.equal(run(top_p=0.9, temperature=1.3), run(top_p=0.9, temperature=1.3))
    assert not torch.equal(run(temperature=1.3), run(seed=4, temperature=1.3))
    greedy = kk.generate(model, ids, 24, cuda_graph=False)
    for kw in (dict(top_p=0.0), dict(top_k=1), dict(min_p=1.0), dict(temperature=0.0)):
        assert torch.equal(run(**kw), greedy), kw
    got = run(top_k=3, top_p=0.8, min_p=0.01)
    cache = kk.KushHFCache(model.config, max_length=64)
    logits = model(ids, past_key_values=cache, use_cache=True).logits[:, -1]
    g = torch.Generator(DEV).manual_seed(3)
    for i in range(24):
        u = torch.rand(2, device=DEV, generator=g)
        tok = kk.sample(logits, u, top_k=3, top_p=0.8, min_p=0.01)
        assert torch.equal(tok, got[:, 40 + i]), i
        logits = model(tok[:, None], past_key_values=cache, use_cache=True).logits[:, -1]
