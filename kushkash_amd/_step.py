"""What surrounds the attention of a serving step, on the GPU kernels of csrc/kush_step.hip (include/kushkash_amd_step.h):
its index arrays -- a decode step's block table, a prefill step's maps -- built from the requests' lengths, and the next
tokens, drawn from the logits and given random numbers. On other devices block_table and step_maps are torch operations
of the same results (the serving integrations' host path runs on block_table; its maps are numpy's); sample is for the GPU."""
from __future__ import annotations

from dataclasses import dataclass, replace

import torch

from . import _lib
from ._window import PAGE, check_limit, pages_left_out

_INDEX = (torch.int32, torch.int64)
MOST_REQUESTS = 1 << 16


def _call(name: str, device: torch.device, *args) -> None:
    with torch.cuda.device(device):
        _lib.call(name, *args, torch.cuda.current_stream(device).cuda_stream)


def _native(name: str, first: torch.Tensor, *args):
    """The call's result in native code, or None: not taken, nothing was launched."""
    m = _lib.native()
    return None if m is None else getattr(m, name)(first, *args, torch._C._cuda_getCurrentRawStream(first.get_device()))


def _index(name: str, t: torch.Tensor, n: int, device: torch.device, dtypes=(torch.int32,)) -> None:
    if t.dtype not in dtypes or not t.is_contiguous() or t.dim() != 1 or t.numel() != n or t.device != device:
        raise ValueError(f"{name} must be contiguous {' or '.join(str(d).split('.')[1] for d in dtypes)} [{n}] on {device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _map(name: str, t: torch.Tensor, rows: int | None, device: torch.device) -> None:
    if t.dtype != torch.int32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or t.device != device:
        raise ValueError(f"{name} must be int32 [rows, columns] with unit column stride on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    if rows is not None and t.shape[0] < rows:
        raise ValueError(f"{name} needs a row per request ({rows}), got {t.shape[0]}")


# ------------------------------------------------------------------ block tables
def block_table(req_to_token: torch.Tensor, req: torch.Tensor, seq_lens: torch.Tensor, pages: int,
                out: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(block table [R, pages], seq_lens [R], slots [R]), int32, of R requests: an engine's token map req_to_token (int32
    [map rows, context], a token's slot being its block * 32 + its row in the page) read at rows req [R] for the pages
    that seq_lens [R] (both int32 or int64) reach; 0 behind them, and where req or a length is outside the map. slots is
    req. out: the three arrays to fill (a captured step's static buffers; the table's rows may be strided)."""
    if req_to_token.is_cuda and (got := _native("block_table", req_to_token, req, seq_lens, pages, out)) is not None:
        return got
    dev, R = req_to_token.device, req.numel()
    _map("req_to_token", req_to_token, None, dev)
    _index("req", req, R, dev, _INDEX)
    _index("seq_lens", seq_lens, R, dev, _INDEX)
    if pages < 0 or pages > 65535 * 256:
        raise ValueError(f"pages must be 0 .. {65535 * 256}, got {pages}")
    if out is None:
        out = (torch.empty(R, pages, dtype=torch.int32, device=dev),
               *(torch.empty(R, dtype=torch.int32, device=dev) for _ in range(2)))
    table, lens, slots = out
    _map("out[0]", table, None, dev)
    if table.shape != (R, pages) or (R > 1 and table.stride(0) < pages):
        raise ValueError(f"out[0] must be [{R}, {pages}] with rows apart, got {tuple(table.shape)}")
    _index("out[1]", lens, R, dev)
    _index("out[2]", slots, R, dev)
    if dev.type != "cuda":
        n = seq_lens.long().clamp(max=req_to_token.shape[1])
        known = (req >= 0) & (req < req_to_token.shape[0])
        first = req_to_token[:, ::PAGE][:, :pages]                  # each page's first token
        cols = first.shape[1]
        if first.numel():
            seen = (torch.arange(cols) * PAGE < n[:, None]) & known[:, None]
            ids = torch.div(first[torch.where(known, req, 0).long()], PAGE, rounding_mode="floor")
            table[:, :cols].copy_(torch.where(seen, ids, 0))
        else:
            cols = 0
        table[:, cols:].zero_()
        lens.copy_(seq_lens)
        slots.copy_(req)
    elif R:
        _call("kush_block_table", dev, req_to_token.data_ptr(), req_to_token.stride(0), *req_to_token.shape, req.data_ptr(),
              int(req.dtype == torch.int64), seq_lens.data_ptr(), int(seq_lens.dtype == torch.int64), R, pages,
              table.data_ptr(), max(table.stride(0), pages), lens.data_ptr(), slots.data_ptr())
    return out


# ------------------------------------------------------------------ maps of a prefill step
@dataclass(frozen=True)
class MapSizes:
    """The sizes of a step's maps, and the window they are for (map_sizes)."""
    requests: int
    tokens: int
    keys: int
    jobs: int
    pages: int
    tails: int
    window: int = 0
    sinks: int = 0

    def __post_init__(self):
        object.__setattr__(self, "numbers", (self.requests, self.tokens, self.keys, self.jobs, self.pages, self.tails,
                                             self.window, self.sinks))

    def writes(self) -> "MapSizes":
        """The sizes without the maps that unpack history: of a step that only writes its tokens."""
        return replace(self, pages=0, tails=0)

    def times(self, n: int) -> "MapSizes":
        """The sizes of n steps of these one behind the other: of sequences of one length each."""
        return MapSizes(*(n * x for x in self.numbers[:-2]), self.window, self.sinks)


@dataclass
class StepMaps:
    """A prefill step's index arrays (step_maps), int32 but for slot_map (int64), in request order."""
    q_start: torch.Tensor      # [R + 1] running sum of the new tokens
    key_start: torch.Tensor    # [R + 1] running sum of the keys: kept history, then new tokens
    seq_lens: torch.Tensor     # [R] history + new tokens
    job_seq: torch.Tensor      # [jobs] request,
    job_page: torch.Tensor     # [jobs]   and logical page, of every page that new tokens touch (Ops.write)
    page_blk: torch.Tensor     # [pages] block,
    page_dst: torch.Tensor     # [pages]   and first key row, of every full page of kept history (Ops.unpack)
    tail_blk: torch.Tensor     # [tails] block of a history's unfinished page,
    tail_info: torch.Tensor    # [tails, 3]   its first key row, tokens and tail slot
    new_dst: torch.Tensor      # [tokens] key row of every new token
    slot_map: torch.Tensor     # [tokens] its block * 32 + its row in the page
    sizes: MapSizes


def map_sizes(new_tokens, history, *, window: int | None = None, sinks: int = 0) -> MapSizes:
    """The sizes of step_maps' arrays for requests of these lengths (sequences of integers on the host). With a window the
    history's pages between the sinks and the window of each request's first new token are left out of the keys."""
    window, sinks = check_limit(window, sinks)
    t, h = [int(x) for x in new_tokens], [int(x) for x in history]
    if len(t) != len(h) or any(x < 0 for x in t + h):
        raise ValueError("new_tokens and history need one length >= 0 per request")
    if len(t) > MOST_REQUESTS:
        raise ValueError(f"at most {MOST_REQUESTS} requests, got {len(t)}")
    gap = [pages_left_out(x, window, sinks) for x in h] if window else [0] * len(h)
    size = MapSizes(len(t), sum(t), sum(t) + sum(h) - PAGE * sum(gap),
                    sum((b + a - 1) // PAGE - b // PAGE + 1 for a, b in zip(t, h) if a),
                    sum(b // PAGE for b in h) - sum(gap), sum(b % PAGE != 0 for b in h), window, sinks)
    if max(size.keys, size.tokens, max((a + b for a, b in zip(t, h)), default=0)) >= 1 << 31:
        raise ValueError("a step's keys must stay below 2^31")
    return size


_MAPS = (("q_start", "requests", 1, 1), ("key_start", "requests", 1, 1), ("seq_lens", "requests", 0, 1),
         ("job_seq", "jobs", 0, 1), ("job_page", "jobs", 0, 1), ("page_blk", "pages", 0, 1), ("page_dst", "pages", 0, 1),
         ("tail_blk", "tails", 0, 1), ("tail_info", "tails", 0, 3), ("new_dst", "tokens", 0, 1))


def step_maps(new_tokens: torch.Tensor, history: torch.Tensor, slots: torch.Tensor, block_table: torch.Tensor,
              sizes: MapSizes) -> StepMaps:
    """The index arrays of a prefill step whose request r adds new_tokens[r] tokens to history[r] cached ones, its exact K
    tail in slot slots[r] (int32 [R]) and its pages in block_table[r] (int32 [R, pages]): what Ops.write, Ops.unpack and the
    ragged attention of the step take. sizes: map_sizes of the same lengths, which the host knows before the step. Lengths
    on the device that need more than the sizes hold are cut off at them."""
    if new_tokens.is_cuda and (got := _native("step_maps", new_tokens, history, slots, block_table, sizes.numbers)) is not None:
        return StepMaps(*got, sizes)
    dev, R = new_tokens.device, sizes.requests
    for name, t in (("new_tokens", new_tokens), ("history", history), ("slots", slots)):
        _index(name, t, R, dev)
    _map("block_table", block_table, R, dev)
    at, cuts = 0, []
    for name, count, more, width in _MAPS:
        n = (getattr(sizes, count) + more) * width
        cuts.append((name, at, n, width))
        at += n
    at += at & 1                                                    # the int64 map behind them, 8-byte aligned
    buf = torch.empty(at + 2 * sizes.tokens, dtype=torch.int32, device=dev)
    maps = StepMaps(**{name: buf[a:a + n].view(-1, 3) if width == 3 else buf[a:a + n] for name, a, n, width in cuts},
                    slot_map=buf[at:].view(torch.int64), sizes=sizes)
    if R == 0:
        buf.zero_()
    elif dev.type != "cuda":
        _host_maps(maps, new_tokens, history, slots, block_table, sizes)
    else:
        _call("kush_step_maps", dev, new_tokens.data_ptr(), history.data_ptr(), slots.data_ptr(), block_table.data_ptr(),
              block_table.stride(0), block_table.shape[1], R, sizes.window, sizes.sinks, sizes.jobs, sizes.pages, sizes.tails,
              sizes.tokens, *(buf.data_ptr() + 4 * a for _, a, _, _ in cuts), buf.data_ptr() + 4 * at)
    return maps


def _host_maps(m: StepMaps, new_tokens, history, slots, block_table, sizes: MapSizes) -> None:
    """step_maps on the CPU (lengths that agree with the sizes)."""
    t, h = new_tokens.long(), history.long()
    first = -(-sizes.sinks // PAGE)
    gap = ((h - sizes.window + 1).clamp(min=0) // PAGE - first).clamp(min=0) if sizes.window else torch.zeros_like(h)
    kept, full = h - PAGE * gap, h // PAGE
    for out, x in ((m.q_start, t), (m.key_start, kept + t)):
        out[0] = 0
        out[1:] = torch.cumsum(x, 0)
    m.seq_lens.copy_(h + t)

    def runs(counts):
        r = torch.repeat_interleave(torch.arange(len(counts)), counts)
        return r, torch.arange(len(r)) - (torch.cumsum(counts, 0) - counts)[r]

    r, i = runs(torch.where(t > 0, (h + t - 1) // PAGE - full + 1, 0))
    m.job_seq.copy_(r)
    m.job_page.copy_(full[r] + i)
    r, i = (x[:sizes.pages] for x in runs(full - gap))
    m.page_blk.copy_(block_table[r, torch.where(i < first, i, i + gap[r])])
    m.page_dst.copy_(m.key_start[r] + PAGE * i)
    r = runs((h % PAGE > 0).long())[0][:sizes.tails]
    m.tail_blk.copy_(block_table[r, full[r]])
    m.tail_info.copy_(torch.stack([m.key_start[r] + PAGE * (full - gap)[r], h[r] % PAGE, slots[r].long()], 1))
    r, i = runs(t)
    m.new_dst.copy_(m.key_start[r] + kept[r] + i)
    m.slot_map.copy_(block_table[r, (h[r] + i) // PAGE].long() * PAGE + (h[r] + i) % PAGE)


# ------------------------------------------------------------------ sampling
_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _setting(name: str, x, rows: int, device: torch.device, dtype: torch.dtype, low: float, high: float):
    """(value for all rows, address of one per row or None)"""
    if isinstance(x, torch.Tensor):
        _index(name, x, rows, device, (dtype,))
        return (0 if dtype == torch.int32 else 0.0), x.data_ptr()
    if dtype == torch.int32:
        if isinstance(x, bool) or not isinstance(x, int):
            raise ValueError(f"{name} must be an integer or an int32 tensor, got {x!r}")
    else:
        x = float(x)
    if not low <= x <= high:
        raise ValueError(f"{name} must be {low} .. {high}, got {x}")
    return x, None


def sample(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row of logits [B, V] (fp32, fp16 or bf16) and random number uniforms [B] (fp32 in [0, 1)); int64 [B].
    With a row's tokens in the order of (logit descending, index ascending) and weights w = exp((logit - largest) /
    temperature):
        top_k > 0    the first top_k are kept;
        top_p < 1    of those, the tokens that have less than top_p of their mass before them;
        min_p > 0    of those, the tokens with w >= min_p;
    the first token always. The token is the first index whose running sum of kept weights, in the vocabulary's order,
    exceeds the random number times the sum of all (1 and more: the last kept one; NaN and less than 0 count as 0): the same for
    the same inputs, on every call. temperature 0 takes the first of the order. A row with a NaN, or without a logit above -inf, gives -1. Each setting is a number, or a tensor
    with one per row (fp32; top_k int32). Weights are held in multiples of 2^-min(50, 63 - log2 V) of the largest, one at least: for
    up to 2^19 tokens the sum of all is off by less than 2^-24 of it, at 2^24 by 2^-15. On the GPU."""
    if logits.is_cuda and (got := _native("sample", logits, uniforms, temperature, top_k, top_p, min_p, out)) is not None:
        return got
    if logits.dim() != 2 or logits.dtype not in _CODE or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"logits must be fp32, fp16 or bf16 [rows, vocabulary] with unit column stride, got {logits.dtype} "
                         f"{tuple(logits.shape)}")
    B, V = logits.shape
    dev = logits.device
    if dev.type != "cuda":
        raise ValueError("sample runs on the GPU (logits on a 'cuda' device under ROCm)")
    if not 1 <= V <= 1 << 24 or (B > 1 and logits.stride(0) < 0):
        raise ValueError(f"the vocabulary must have 1 .. 2^24 tokens, got {V}")
    if torch.is_grad_enabled() and logits.requires_grad:
        raise ValueError("sample has no derivative: detach the logits")
    _index("uniforms", uniforms, B, dev, (torch.float32,))
    inf = float("inf")
    settings = (*_setting("temperature", temperature, B, dev, torch.float32, 0.0, 1e30),
                *_setting("top_k", top_k, B, dev, torch.int32, 0, 2 ** 31 - 1),
                *_setting("top_p", top_p, B, dev, torch.float32, 0.0, inf),
                *_setting("min_p", min_p, B, dev, torch.float32, 0.0, inf))
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    _index("out", out, B, dev, (torch.int64,))
    if B:
        scratch = torch.empty(_lib.lib().kush_sample_scratch(B, V), dtype=torch.uint8, device=dev)
        _call("kush_sample", dev, _CODE[logits.dtype], logits.data_ptr(), logits.stride(0) if B > 1 else V, B, V,
              uniforms.data_ptr(), *settings, out.data_ptr(), scratch.data_ptr(), scratch.numel())
    return out
