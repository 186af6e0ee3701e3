"""generate over logits that hold no distribution: an error that names the rows, and no id outside the vocabulary on the way to it."""
import pytest
import torch

import kushkash_amd as kk
from kushkash_amd._generate import EOS_LAG, _StopSignal

pytestmark = pytest.mark.gpu
transformers = pytest.importorskip("transformers")
DEV = "cuda"


def model():
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    m = LlamaForCausalLM(LlamaConfig(vocab_size=256, hidden_size=256, intermediate_size=512, num_attention_heads=4,
                                     num_key_value_heads=2, head_dim=64, num_hidden_layers=1)).to(DEV, torch.bfloat16).eval()
    m.seen = []

    def look(_, args):                                       # the ids that the embedding is given
        if not torch.cuda.is_current_stream_capturing():
            m.seen.append((int(args[0].min()), int(args[0].max())))
    m.model.embed_tokens.register_forward_pre_hook(look)
    return m


def break_rows(m, rows, value, after):
    """Logits of `rows` all `value` from the forward after `after` others on."""
    calls = []

    def hook(_, args, out):
        calls.append(0)
        if len(calls) > after:
            out[rows] = value
        return out
    m.lm_head.register_forward_hook(hook)


def run(m, n, **kw):
    ids = torch.randint(0, 256, (3, 20), generator=torch.Generator().manual_seed(1)).to(DEV)
    return kk.generate(m, ids, n, do_sample=True, **kw)


@pytest.mark.parametrize("value", [float("nan"), float("-inf")])
@pytest.mark.parametrize("after", [0, 1, 4])
@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(min_p=0.1, top_k=20, eos_token_id=[300, 301]),
                                dict(generator=True, eos_token_id=300)], ids=str)
def test_rows_without_a_distribution_end_the_run(value, after, kw):
    m = model()
    break_rows(m, [0, 2], value, after)
    if "generator" in kw:
        kw = dict(kw, generator=torch.Generator(device=DEV).manual_seed(3))
    with pytest.raises(RuntimeError, match=r"rows \[0, 2\]"):
        run(m, 40, cuda_graph=False, **kw)
    assert len(m.seen) <= after + 2 + EOS_LAG + 1 and all(0 <= a and b < 256 for a, b in m.seen)
    for n in range(after + 1, 3):                            # ends before the flags come round
        m = model()
        break_rows(m, [0, 2], value, after)
        with pytest.raises(RuntimeError, match=r"rows \[0, 2\]"):
            run(m, n, cuda_graph=False, **kw)


def test_replayed_steps():
    m = model()
    with torch.no_grad():
        m.lm_head.weight[5].fill_(float("nan"))
    with pytest.raises(RuntimeError, match=r"rows \[0, 1, 2\]"):
        run(m, 30, top_p=0.9, cuda_graph=True)


def test_rows_that_are_done_may_break():
    """A row that has ended keeps emitting EOS whatever its logits are, and the others go on."""
    m = model()
    calls = []

    def hook(_, args, out):
        calls.append(0)
        out[1] = float("nan") if len(calls) > 1 else torch.where(torch.arange(256, device=DEV) == 9, 50.0, -50.0).to(out.dtype)
        out[0, :, 9] = out[2, :, 9] = float("-inf")
        return out
    m.lm_head.register_forward_hook(hook)
    out = run(m, 12, top_p=0.9, eos_token_id=9, cuda_graph=False)
    assert out.shape == (3, 32) and (out[1, 20:] == 9).all() and not (out[[0, 2], 20:] == 9).any() and (out >= 0).all()


def test_sound_rows_give_what_they_gave():
    """The draws are the sampling kernel's on the model's logits, step for step, with EOS and without."""
    outs = []
    for kw in (dict(), dict(eos_token_id=300)):
        torch.manual_seed(7)
        outs.append(run(model(), 16, top_p=0.8, cuda_graph=False, **kw))
    assert torch.equal(*outs) and int(outs[0].min()) >= 0


def test_the_flags_of_a_step():
    s = _StopSignal(torch.tensor([4], device=DEV), 2, torch.device(DEV))
    tok = s.mask(s.admit(torch.tensor([3, -1], device=DEV)))
    assert tok.tolist() == [3, 0]
    for i in range(1, EOS_LAG + 1):
        assert s.finished(tok, i) is False
    with pytest.raises(RuntimeError, match=r"rows \[1\]"):
        s.finished(tok, EOS_LAG + 1)
