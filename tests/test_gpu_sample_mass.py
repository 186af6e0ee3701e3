"""sample where the kept mass is large or many tiny weights add up: random numbers at and past the ends of their range over flat
rows, and vocabularies whose tokens of next to no weight must not weigh anything together. Whole numbers, equal to the definition in
64 bits."""
import pytest
import torch

import kushkash_amd as kk
from test_gpu_sample import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def flat(V, top, seed=0):
    """Rows with `top` equal largest logits: the first ones, the last ones, scattered ones; the others 3 below and masked."""
    g = torch.Generator().manual_seed(seed)
    x = torch.full((6, V), -3.0)
    x[3:] = float("-inf")
    for r in range(6):
        at = (torch.arange(top), V - 1 - torch.arange(top), torch.randperm(V, generator=g)[:top])[r % 3]
        x[r, at] = 1.5
    return x


@pytest.mark.parametrize("u", [1.0, 2.0, float("inf"), 1 - 2.0 ** -24, 0.5, 0.0, -1.0])
@pytest.mark.parametrize("V, top", [(64, 64), (1000, 64), (4096, 4096), (4097, 64), (8000, 50), (8000, 64), (8000, 300), (8000, 1900),
                                    (8000, 3000), (8000, 8000), (30011, 50), (30011, 9000), (30011, 30011)])
def test_random_numbers_over_flat_rows(V, top, u):
    """A random number of 1 or more takes the last kept token, whichever way the list goes; below 0 counts as 0. 64 equal weights
    pass 2^53, where a 64-bit float no longer holds a mass less one."""
    x, us = flat(V, top, seed=V + top), torch.full((6,), u)
    for setting in (dict(), dict(k=top), dict(k=max(1, top - 3)), dict(p=0.75), dict(k=top, p=0.5, m=0.01)):
        # (the definition is taken at the ends of the range that random numbers have)
        want = torch.full((6,), min(max(u, 0.0), 1.0))
        got = kk.sample(x.to(DEV), us.to(DEV), temperature=1.0, top_k=setting.get("k", 0), top_p=setting.get("p", 1.0),
                        min_p=setting.get("m", 0.0))
        assert torch.equal(got, kk.sample(x.to(DEV), want.to(DEV), temperature=1.0, top_k=setting.get("k", 0),
                                          top_p=setting.get("p", 1.0), min_p=setting.get("m", 0.0)))
        check(x, want, **setting)


def test_a_random_number_that_is_none():
    x = flat(8000, 64)
    assert torch.equal(kk.sample(x.to(DEV), torch.full((6,), float("nan")).to(DEV), top_k=64),
                       kk.sample(x.to(DEV), torch.zeros(6).to(DEV), top_k=64))


@pytest.mark.parametrize("V", [151936, 262208, 1 << 19])
def test_tokens_of_next_to_no_weight(V):
    """One token next to all others at e^-100 of its weight: they have 2e-38 of the mass together, so the smallest random number
    above 0 takes the one. (A weight above 0 is held as one unit at least, 2^-44 at 2^19 tokens: 2^-25 of the mass together,
    below the smallest random number, 2^-24.)"""
    x = torch.full((2, V), -100.0)
    x[0, V - 1] = x[1, V // 2] = 0.0
    for u in (2.0 ** -24, 0.25, 1 - 2.0 ** -24):
        want = [V - 1, V // 2]
        for kw in (dict(), dict(top_p=0.999999), dict(top_k=V - 1)):
            got = kk.sample(x.to(DEV), torch.full((2,), u).to(DEV), **kw).tolist()
            assert got == want, (u, kw)
