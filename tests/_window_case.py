"""Inputs and 64-bit references of the attention under a window (the query at position p sees key j <= p when
j > p - window or j < sinks), shared by its tests. The references go token by token through the definition."""
import torch

from kushkash_amd import record_bytes
from kushkash_amd._records import dequant_records

PAGE = 32


def seen(p: int, window: int, sinks: int) -> list[int]:
    return [j for j in range(p + 1) if j > p - window or j < sinks]


def paged(lens, D, bits, H, dtype, seed, device="cpu"):
    """A cache of random records for sequences of these lengths: dict of records, block table (blocks in random order),
    seq_lens, tail_idx (slots in random order) and tail_k. V within about +-3, K about +-3 with a bias per channel."""
    g = torch.Generator().manual_seed(seed)
    S = len(lens)
    wide = max(1, -(-max(lens, default=0) // PAGE))
    blocks = S * wide + 2
    body = 2 * PAGE * (D if bits == 8 else D // 2)
    step = 2.0 / (8 if bits == 4 else 128)
    rec = torch.randint(0, 256, (blocks, H, record_bytes(D, bits)), generator=g, dtype=torch.uint8)
    meta = torch.empty(blocks, H, 2 * D + 2 * PAGE, dtype=torch.float16)
    meta[..., :D] = step * (0.5 + torch.rand(blocks, H, D, generator=g))
    meta[..., D:2 * D] = 0.3 * torch.randn(H, D, generator=g) + 0.1 * torch.randn(blocks, H, D, generator=g)
    meta[..., 2 * D:2 * D + PAGE] = step * (0.5 + torch.rand(blocks, H, PAGE, generator=g))
    meta[..., 2 * D + PAGE:] = 0.2 * torch.randn(blocks, H, PAGE, generator=g)
    rec[..., body:] = meta.view(torch.uint8)
    table = (torch.randperm(blocks - 2, generator=g)[:S * wide].view(S, wide) + 1).to(torch.int32)
    c = dict(records=rec, table=table, lens=torch.tensor(lens, dtype=torch.int32),
             tidx=torch.randperm(S + 2, generator=g)[:S].to(torch.int32),
             tail=torch.randn(S + 2, H, PAGE, D, generator=g).to(dtype))
    return {k: v.to(device) for k, v in c.items()}


def decode_reference(q, c, D, bits, G, scale, window, sinks):
    """[S, Hq, D] in 64 bits, and the largest |value| that any query sees."""
    H = c["tail"].shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    most = 0.0
    rec, table, tail = c["records"].cpu(), c["table"].cpu().long(), c["tail"].cpu().double()
    for s, n in enumerate(c["lens"].cpu().tolist()):
        js = torch.tensor(seen(n - 1, window, sinks), dtype=torch.long)
        if not len(js):
            continue
        kp, vp = dequant_records(rec[table[s, js // PAGE]], D, bits, torch.float64)       # [tokens, H, 32, D]: a page each
        at = (js % PAGE).view(-1, 1, 1, 1).expand(-1, H, 1, D)
        K, V = (x.gather(2, at)[:, :, 0] for x in (kp, vp))
        part = js >= n // PAGE * PAGE
        if n % PAGE:
            K[part] = tail[int(c["tidx"][s])][:, js[part] % PAGE].transpose(0, 1)
        most = max(most, float(V.abs().max()))
        for h in range(H):
            qs = q[s, h * G:(h + 1) * G].double().cpu()
            out[s, h * G:(h + 1) * G] = torch.softmax(scale * qs @ K[:, h].T, -1) @ V[:, h]
    return out, most


def rows_reference(q, k, v, scale, window, sinks):
    """window_attention of q [T, Hq, D] over k, v [N, Hk, D] in 64 bits."""
    T, Hq, D = q.shape
    N, G = k.shape[0], Hq // k.shape[1]
    at, j = torch.arange(N - T, N)[:, None], torch.arange(N)[None, :]
    hidden = (j > at) | ((j <= at - window) & (j >= sinks))
    out = torch.empty(q.shape, dtype=torch.float64)
    for i in range(Hq):
        s = (scale * q[:, i].double() @ k[:, i // G].double().T).masked_fill(hidden, float("-inf"))
        out[:, i] = torch.softmax(s, -1) @ v[:, i // G].double()
    return out


def half_step(dtype) -> float:
    """The largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2
