"""Attention limited to a window of the last tokens and a few first ones (sinks) that stay visible: the query at
position p sees key j <= p when j > p - window or j < sinks. The cache's decode takes the limit as Ops.decode(window=,
sinks=); window_attention is the same limit on rows, for prompts and chunks. Kernels: csrc/kush_decode.h and
csrc/kush_attend.h (include/kushkash_amd_window.h)."""
from __future__ import annotations

from itertools import accumulate

import torch

from . import _attend

PAGE = 32
MOST = 1 << 30                    # window and sinks at most


def check_limit(window: int | None, sinks: int) -> tuple[int, int]:
    """(window, sinks) as the kernels take them, (0, 0) for no window. ValueError for anything else than a window of at
    least one token (the query's own) and sinks of at least none, or for sinks without a window."""
    if window is None:
        if sinks:
            raise ValueError("sinks are for attention with a window (window=None sees every token)")
        return 0, 0
    for name, x, least in (("window", window, 1), ("sinks", sinks, 0)):
        if isinstance(x, bool) or not isinstance(x, int) or not least <= x <= MOST:
            raise ValueError(f"{name} must be an integer of {least} .. 2^30, got {x!r}")
    return window, sinks


def pages_left_out(position: int, window: int, sinks: int) -> int:
    """Pages that the query at `position` sees nothing of between the sinks' pages and its window's."""
    return max(0, max(0, position - window + 1) // PAGE - -(-sinks // PAGE)) if window else 0


def _products(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int, scale: float,
              block_bytes: int = 1 << 28) -> torch.Tensor:
    """q [B, T, Hq, D] over k, v [B, N, Hk, D] by fp32 products, as many queries at a time as keep the scores and their
    exponentials within block_bytes (one at least). Differentiable."""
    B, T, Hq, D = q.shape
    N, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    kt, vt = (x.transpose(1, 2).float() for x in (k, v))                     # [B, Hk, N, D]
    step = T
    while step > 1 and 8 * B * Hq * step * min(N, window + sinks + step) > block_bytes:
        step //= 2
    out = []
    for a in range(0, T, step):
        b = min(T, a + step)
        at = torch.arange(N - T + a, N - T + b, device=q.device)[:, None]
        low = max(0, N - T + a - window + 1)
        key = torch.arange(low, N - T + b, device=q.device)
        if sinks and low:
            key = torch.cat([torch.arange(min(sinks, low), device=q.device), key])
        qf = q[:, a:b].float().transpose(1, 2).reshape(B, Hk, G * (b - a), D)
        hidden = ((key > at) | ((key <= at - window) & (key >= sinks))).repeat(G, 1)
        s = (torch.matmul(qf, kt[:, :, key].transpose(-1, -2).contiguous()) * scale).masked_fill(hidden, float("-inf"))
        o = torch.matmul(torch.softmax(s, -1), vt[:, :, key])
        out.append(o.view(B, Hq, b - a, D).transpose(1, 2))
    return torch.cat(out, 1).to(q.dtype)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int, sinks: int = 0,
                     scale: float | None = None, cu: tuple[torch.Tensor, torch.Tensor] | None = None,
                     spans: list[tuple[int, int]] | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the last T of N positions, each query limited to the last `window` keys up to its own and the
    first `sinks`: q [B, T, Hq, D] over k, v [B, N, Hk, D], N >= T (q head i reads kv head i // (Hq / Hk)). Returns q's
    shape and dtype, in `out` where given.

    spans = [(T, N), ..]: sequences of these lengths packed end to end in q [rows, Hq, D] and k, v [rows, Hk, D]; cu =
    (cu_q, cu_k), their running sums as int32 device tensors [sequences + 1] (built from spans where not given, which
    copies them to the device).

    bf16 and fp16 rows of head_dim 64, 128 and 256 on the GPU, 16-byte aligned, run on the prefill attention kernel
    (forward only); anything else (fp32, other sizes, the CPU, inputs that ask for derivatives) in fp32 products. Keys
    may be left out of the rows between the sinks and the first query's window, if whole: positions count in the rows
    given. Keys that a row does not see may be infinite or NaN. Their values may not, as a weight of zero times them is NaN;
    those at least 64 rows from what any query of the sequence sees are not read."""
    window, sinks = check_limit(window, sinks)
    if window == 0:
        raise ValueError("window_attention needs a window")
    return limited_attention(q, k, v, window, sinks, scale, cu, spans, out)


def limited_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int, scale: float | None = None,
                      cu=None, spans=None, out: torch.Tensor | None = None, block_bytes: int = 1 << 28) -> torch.Tensor:
    """window_attention of a checked limit, its scratch (partials of split keys, or scores) within block_bytes."""
    if (o := _attend.window_native(q, k, v, q.shape[-1] ** -0.5 if scale is None else scale, cu, spans, out, window, sinks,
                                   block_bytes)) is not None:
        return o
    packed = spans is not None
    rank = 3 if packed else 4
    if any(x.dim() != rank for x in (q, k, v)):
        raise ValueError("q, k and v must be [rows, heads, dim] with spans, [batch, rows, heads, dim] without")
    if cu is not None and not packed:
        raise ValueError("cu needs spans, the sequences' lengths on the host")
    if k.shape != v.shape or q.shape[-1] != k.shape[-1] or not k.shape[-2] or q.shape[-2] % k.shape[-2] or not q.shape[-1]:
        raise ValueError(f"k and v must have one shape, q their head_dim and a multiple of their heads: got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype) or not q.is_floating_point():
        raise ValueError(f"q, k and v must have one floating-point dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    if not (q.device == k.device == v.device):
        raise ValueError(f"q, k and v must be on one device, got {q.device}, {k.device}, {v.device}")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if packed:
        spans = [(int(t), int(n)) for t, n in spans]
        if any(t < 0 or n < t for t, n in spans):
            raise ValueError("every sequence needs as many keys as queries, or more (N >= T >= 0)")
        if sum(t for t, _ in spans) != q.shape[0] or sum(n for _, n in spans) != k.shape[0]:
            raise ValueError(f"spans hold {sum(t for t, _ in spans)} queries and {sum(n for _, n in spans)} keys, the rows "
                             f"{q.shape[0]} and {k.shape[0]}")
        if cu is not None:
            for x in cu:
                if x.dtype != torch.int32 or not x.is_contiguous() or x.numel() != len(spans) + 1 or x.device != q.device:
                    raise ValueError(f"cu must be two contiguous int32 tensors of {len(spans) + 1} entries on {q.device}")
    elif q.shape[0] != k.shape[0] or k.shape[1] < q.shape[1]:
        raise ValueError(f"k and v need q's batch and as many rows or more, got {tuple(q.shape)} and {tuple(k.shape)}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device):
        raise ValueError("out must have q's shape, dtype and device")
    if q.numel() == 0:
        return torch.empty_like(q) if out is None else out
    if _attend.takes(q, k, v, scale):
        dst = out if out is not None and _attend.takes_out(out) else None
        if packed:
            if cu is None:
                cu = tuple(torch.tensor([0, *accumulate(s[i] for s in spans)], dtype=torch.int32, device=q.device) for i in (0, 1))
            cu = (*cu, max(t for t, _ in spans), max(n for _, n in spans))
        o = _attend.attend(q, k, v, True, scale, cu=cu, spans=spans, out=dst, scratch=block_bytes, window=window, sinks=sinks)
        return o if out is None or dst is not None else out.copy_(o)
    if not packed:
        o = _products(q, k, v, window, sinks, scale, block_bytes)
    else:
        parts, a, c = [], 0, 0
        for t, n in spans:
            if t:
                parts.append(_products(q[None, a:a + t], k[None, c:c + n], v[None, c:c + n], window, sinks, scale,
                                       block_bytes)[0])
            a, c = a + t, c + n
        o = torch.cat(parts)
    return o if out is None else out.copy_(o)
