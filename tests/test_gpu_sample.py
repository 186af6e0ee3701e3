"""sample on the GPU against its definition in 64 bits: whole numbers, equal."""
import numpy as np
import pytest
import torch

import kushkash_amd as kk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def reference(x, u, T, k, p, m):
    """One row: the token, by the definition. Python integers and 64-bit floats."""
    x = np.asarray(x, dtype=np.float64)
    if np.isnan(x).any() or not (x > -np.inf).any():
        return -1
    order = np.lexsort((np.arange(len(x)), -x))
    if T == 0:
        return int(order[0])
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / T))
    rank = np.empty(len(x), dtype=np.int64)
    rank[order] = np.arange(len(x))
    if 0 < k < len(x):
        w = np.where(rank < k, w, 0.0)
    run = np.cumsum(w[order])
    before = np.empty(len(x))
    before[order] = run - w[order]
    keep = np.ones(len(x), dtype=bool)
    if p < 1:
        keep &= before < p * run[-1]
    keep &= w >= m
    keep[order[0]] = True
    w = np.where(keep, w, 0.0)
    run = np.cumsum(w)
    return int(np.argmax(run > u * run[-1])) if u < 1 else int(np.flatnonzero(w)[-1])


def check(x, u, T=1.0, k=0, p=1.0, m=0.0):
    def at(s, i):
        return s[i].item() if isinstance(s, torch.Tensor) else s
    got = kk.sample(x.to(DEV), u.to(DEV), temperature=T.to(DEV) if isinstance(T, torch.Tensor) else T,
                    top_k=k.to(DEV) if isinstance(k, torch.Tensor) else k, top_p=p.to(DEV) if isinstance(p, torch.Tensor) else p,
                    min_p=m.to(DEV) if isinstance(m, torch.Tensor) else m).tolist()
    want = [reference(x[i].double().numpy(), float(u[i]), at(T, i), at(k, i), at(p, i), at(m, i)) for i in range(len(x))]
    assert got == want


def rand(*shape, seed=0, scale=2.0, dtype=torch.float32):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def uniforms(n, seed=0):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed + 100))


SETTINGS = [dict(), dict(k=1), dict(k=7), dict(k=5000), dict(p=0.9), dict(p=0.0), dict(m=0.05), dict(m=1.0),
            dict(k=50, p=0.8), dict(k=3000, p=0.95, m=0.001), dict(T=0.0), dict(T=0.3, k=40, p=0.9, m=0.01), dict(T=3.0, p=0.99)]


@pytest.mark.parametrize("V", [1, 2, 33, 1000, 4096, 4097, 50257, 151936])
@pytest.mark.parametrize("setting", SETTINGS, ids=str)
def test_settings(V, setting):
    check(rand(5, V, seed=V), uniforms(5, V), **setting)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("setting", SETTINGS, ids=str)
def test_half_precision_logits_tie(dtype, setting):
    """Many equal logits: ties go to the lowest index, also across a cut."""
    check(rand(4, 9001, seed=1, dtype=dtype), uniforms(4, 1), **setting)


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0, 2.0])
def test_the_ends_of_the_random_numbers(u):
    x = rand(3, 7001, seed=2, scale=6.0)
    x[0, :5000] = float("-inf")
    for setting in (dict(), dict(k=9), dict(p=0.7), dict(m=0.1)):
        check(x, torch.full((3,), u), **setting)


@pytest.mark.parametrize("setting", [dict(), dict(k=50), dict(p=0.5), dict(k=9000, p=0.9), dict(k=9000), dict(p=0.9999), dict(k=8500, p=0.3, m=0.9)],
                         ids=str)
def test_lists_that_overflow(setting):
    """Equal logits next to a cut by the ten thousands: the whole row equal, two values, a narrow row."""
    V = 30011
    x = torch.zeros(4, V)
    x[1, ::3] = 0.25
    x[2] = (rand(V, seed=3) * 0.01).to(torch.float16).float()
    x[3, 5:20000] = 4.0
    x[3, 20000:] = float("-inf")
    check(x, uniforms(4, 3), **setting)


def test_rows_without_a_distribution_and_infinities():
    x = rand(6, 513, seed=4)
    x[0] = float("-inf")
    x[1, 77] = float("nan")
    x[2, 400:410] = float("inf")
    x[3] = float("-inf")
    x[3, 300] = -3e38
    x[4, 3] = 3e38
    for setting in (dict(), dict(k=3), dict(p=0.6), dict(T=0.0), dict(k=5, p=0.2, m=0.5)):
        check(x, uniforms(6, 4), **setting)


def test_settings_per_row():
    n = 9
    g = torch.Generator().manual_seed(5)
    T = torch.rand(n, generator=g) + 0.2
    T[3] = 0.0
    k = torch.randint(0, 3000, (n,), generator=g, dtype=torch.int32)
    k[1], k[2] = 0, -4                                                     # off, both
    p = 0.5 + torch.rand(n, generator=g)
    m = 0.1 * torch.rand(n, generator=g)
    check(rand(n, 20011, seed=5), uniforms(n, 5), T=T, k=torch.clamp(k, min=0), p=p, m=m)
    x, u = rand(n, 20011, seed=5).to(DEV), uniforms(n, 5).to(DEV)
    assert torch.equal(kk.sample(x, u, top_k=k.to(DEV)), kk.sample(x, u, top_k=torch.clamp(k, min=0).to(DEV)))


def test_strided_rows_and_many_rows():
    """Rows of a wider buffer (odd strides, unaligned), and more rows than one launch takes."""
    wide = rand(7, 6007, seed=6)
    x, u = wide[1:6:2, 3:5000], uniforms(3, 6)
    want = kk.sample(x.contiguous().to(DEV), u.to(DEV), top_k=20, top_p=0.9)
    assert torch.equal(kk.sample(wide.to(DEV)[1:6:2, 3:5000], u.to(DEV), top_k=20, top_p=0.9), want)
    half = wide.to(torch.bfloat16)
    assert torch.equal(kk.sample(half.to(DEV)[1:6:2, 3:5000], u.to(DEV), top_p=0.9),
                       kk.sample(half[1:6:2, 3:5000].contiguous().to(DEV), u.to(DEV), top_p=0.9))
    x, u = rand(2050, 301, seed=7), uniforms(2050, 7)
    check(x, u, k=20, p=0.9)


def test_the_frequencies_of_a_distribution():
    """Over evenly spread random numbers each token comes up as often as its share says, to one."""
    n = 4096
    x = rand(1, 50, seed=8).expand(n, 50).contiguous()
    u = (torch.arange(n) + 0.5) / n
    got = torch.bincount(kk.sample(x.to(DEV), u.to(DEV)).cpu(), minlength=50)
    share = torch.softmax(x[0].double(), 0) * n
    assert float((got - share).abs().max()) <= 1.0 + 1e-6


def test_replays_of_a_captured_call():
    x, u = rand(6, 30000, seed=9).to(DEV), uniforms(6, 9).to(DEV)
    kk.sample(x, u, top_k=40, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kk.sample(x, u, top_k=40, top_p=0.9)
    for i in range(4):
        x.copy_(rand(6, 30000, seed=20 + i))
        u.copy_(uniforms(6, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kk.sample(x, u, top_k=40, top_p=0.9))


def test_two_streams_at_once():
    x, u = rand(8, 40000, seed=10).to(DEV), uniforms(8, 10).to(DEV)
    want = kk.sample(x, u, top_p=0.8)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [kk.sample(x, u, top_p=0.8) for _ in range(5)]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(t, want) for t in got)


def test_refusals():
    x, u = rand(2, 9).to(DEV), uniforms(2).to(DEV)
    out = torch.empty(2, dtype=torch.int64, device=DEV)
    assert kk.sample(x, u, out=out) is out
    for args, kw in (((x.double(), u), {}), ((x[0], u), {}), ((x.t(), u), {}), ((x, u[:1]), {}), ((x, u.double()), {}),
                     ((x, u.cpu()), {}), ((x.cpu(), u), {}), ((x, u), dict(temperature=-1.0)), ((x, u), dict(temperature=float("nan"))),
                     ((x, u), dict(top_k=-1)), ((x, u), dict(top_k=2.0)), ((x, u), dict(top_k=True)), ((x, u), dict(top_p=-0.1)),
                     ((x, u), dict(min_p=float("nan"))), ((x, u), dict(top_k=u)), ((x, u), dict(top_p=u[:1])),
                     ((x, u), dict(out=out.to(torch.int32))), ((x[:, :0], u), {}), ((x.clone().requires_grad_(), u), {})):
        with pytest.raises(ValueError):
            kk.sample(*args, **kw)
    assert kk.sample(x[:0], u[:0]).shape == (0,)
    with torch.no_grad():
        assert torch.equal(kk.sample(x.clone().requires_grad_(), u), kk.sample(x, u))


@pytest.mark.parametrize("k", [1, 2, 62, 63, 64, 65, 66, 255, 256, 257, 2047, 2048, 2049, 4095, 5200])
@pytest.mark.parametrize("p, m", [(1.0, 0.0), (0.6, 0.0), (0.97, 0.003)])
def test_lists_of_every_length(k, p, m):
    """The list that top-k leaves changes its way at 64 tokens, at a thousand next to a cut, at 2,048 and past 5,120; logits apart,
    equal in pairs, and flat enough that a class holds many."""
    x = torch.cat([rand(2, 9000, seed=k), rand(2, 9000, seed=k + 1, dtype=torch.bfloat16).float(), rand(2, 9000, seed=k, scale=0.01)])
    x[3, ::2] = x[3, 1::2]
    check(x, uniforms(6, k), k=k, p=p, m=m)


@pytest.mark.parametrize("V", [40, 4097])
@pytest.mark.parametrize("setting", [dict(), dict(k=20, p=0.9), dict(p=0.9)], ids=str)
def test_more_rows_than_one_launch_takes(V, setting):
    check(rand(1030, V, seed=V), uniforms(1030, V), **setting)


def test_rows_that_share_their_logits():
    """A row expanded over the batch (stride 0), and rows of a wider array."""
    x, u = rand(1, 5001, seed=3), uniforms(9, 4)
    got = kk.sample(x.to(DEV).expand(9, 5001), u.to(DEV), top_k=60, top_p=0.9).tolist()
    assert got == [reference(x[0].double().numpy(), float(v), 1.0, 60, 0.9, 0.0) for v in u]
    wide = rand(4, 6007, seed=5)
    got = kk.sample(wide.to(DEV)[:, 3:5004], u[:4].to(DEV), top_k=60).tolist()
    assert got == [reference(wide[i, 3:5004].double().numpy(), float(u[i]), 1.0, 60, 1.0, 0.0) for i in range(4)]
