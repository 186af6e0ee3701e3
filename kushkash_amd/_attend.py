"""The prefill attention kernel (csrc/kush_attend.hip, include/kushkash_amd_attend.h): which inputs it takes,
how a call is spread over the chip, and the call. Half-precision rows on the GPU, any batch and row strides,
GQA, causal with the queries at the end of the keys or not, ragged rows packed end to end; forward only.
Reference: the varlen flash attention of kushkash/vllm/backend.py:837-880."""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch

from . import _lib

CUS = 256                        # MI355X compute units
KEYS = 64                        # keys per tile
PARTIAL_BYTES = 1 << 28          # at most this much scratch for split keys
SLOTS = {64: 4 * CUS, 128: 2 * CUS, 256: CUS}       # 4-wave workgroups the chip holds at once, by head_dim
TILE_US = {64: 1.26, 128: 2.14, 256: 2.88}          # a key tile's time with all of them taken
ALONE_US = {64: 0.8, 128: 1.3, 256: 1.9}            # and with a few taken
MERGE_US = 6.0                   # what a second launch adds at least
_Strides = ctypes.c_int64 * 15
# torch.jit.trace, a vmap / grad / functionalize level, and dispatch modes (read on every call)
_tracing, _transform, _modes = (torch._C._get_tracing_state, torch._C._functorch.peek_interpreter_stack,
                                torch._C._len_torch_dispatch_stack)


def _plain(*ts: torch.Tensor) -> bool:
    """Whether the tensors are what a kernel can be handed: no subclass, no tracing or transform around
    them, and no derivative asked for (the kernel has none)."""
    if any(type(t) not in (torch.Tensor, torch.nn.Parameter) for t in ts):
        return False
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        return False
    return not (torch.compiler.is_compiling() or _tracing() is not None or _transform() is not None or _modes()
                or torch.autograd.forward_ad._current_level >= 0)


def _row_strides(t: torch.Tensor, D: int) -> tuple[int, int, int]:
    """(batch, row, head) strides of [.., rows, heads, D]; a dim of one entry counts as packed."""
    st = [0 if t.dim() == 3 or t.shape[0] == 1 else t.stride(0), t.stride(-3), t.stride(-2)]
    if t.shape[-3] == 1:
        st[1] = D
    if t.shape[-2] == 1:
        st[2] = D
    return tuple(st)


def takes(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> bool:
    """Whether the kernel takes q [B, T, Hq, D] (or packed [rows, Hq, D]) over k, v [B, N, Hk, D]: anything
    else is the caller's other paths' (torch's flash kernel, fp32 products)."""
    D = q.shape[-1]
    if (not q.is_cuda or q.dtype not in (torch.bfloat16, torch.float16) or D not in (64, 128, 256)
            or not (k.dtype == v.dtype == q.dtype and k.device == v.device == q.device)
            or not (0.0 < scale < math.inf) or k.shape != v.shape or k.shape[-1] != D or q.dim() != k.dim()
            or (q.dim() == 4 and q.shape[0] != k.shape[0]) or not _plain(q, k, v)):
        return False
    T, Hq, Hk = q.shape[-3], q.shape[-2], k.shape[-2]
    if not q.numel() or not k.numel() or Hq % Hk or T * (Hq // Hk) > 1 << 22 or k.shape[-3] > 1 << 30:
        return False
    for t in (q, k, v):
        st = _row_strides(t, D)
        if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 or s < 0 for s in st):
            return False
        if t is not q and not D <= st[1] <= 1 << 23:
            return False
    return True


def takes_out(out: torch.Tensor) -> bool:
    """Whether the kernel can write this output in place: 16-byte aligned rows, dims adjacent."""
    return (_plain(out) and out.stride(-1) == 1 and out.data_ptr() % 16 == 0
            and not any(s % 8 or s < 0 for s in _row_strides(out, out.shape[-1])))


def window_tiles(window: int, sinks: int, rows: int, group: int) -> int:
    """The most key tiles that a row tile of `rows` rows sees under a window (csrc/kush_attend.hip)."""
    return -(-sinks // KEYS) + (window + (rows - 1) // group) // KEYS + 2


def row_tiles(spans, group: int, waves: int) -> int:
    """Row tiles of all sequences of (T, N) or (T, N, count) together."""
    return sum(-(-s[0] * group // (32 * waves)) * (s[2] if len(s) > 2 else 1) for s in spans)


def plan(spans, group: int, hkv: int, D: int, total_q: int, causal: bool = True,
         scratch: int = PARTIAL_BYTES, window: int = 0, sinks: int = 0) -> tuple[int, int]:
    """(waves, chunk) of a call whose sequences have (T, N, count) query rows and keys. A row tile is 32 waves
    query rows (group heads of each token) of one kv head; 4 waves fill half a CU (a whole one at D 256, a
    quarter at D 64), 8 a whole one.
      8 waves  share each K / V tile among twice the rows, one workgroup to a CU: 1,048 us against 1,097 at 2,048
               tokens x 4 heads over 34,816 keys (8 kv heads, D 128), 3-7 % less from 16,384 keys on at D 64 and 128;
               at 8,192 keys between 2 % more and 4 % less, and 6-20 % more at 2,048. Only where the last round of row
               tiles fills the chip: 3,584 tokens (448 row tiles, 0.88 of two rounds) 1,843 us against 1,996, 3,072
               (384, 0.75) 1,811 against 1,647, 2,176 (272, 0.53) 1,836 against 1,573.
      chunk    split the keys of a row tile where the row tiles leave the chip idle, into as many parts as fill it
               (256 tokens over 8,000 keys: 162 -> 68 us), or, where the longest would run on alone, into
               halves (nine chunks of 61-395 tokens over 800-8,300 keys: 295 -> 268 us), if that gains more than the
               partials cost: half of what the longest row tile is over an even share (the workgroups left have
               more of a CU by then; 0.7 at D 256, one workgroup to a CU) against their bytes out and in at 2.5
               TB/s. The constants are from 700 drawn calls of both sides; without the condition 118 of them were
               2-32 % slower than whole (3,072 tokens over themselves: 101 -> 129 us, 2,048 at D 64: 43 -> 52), with
               it 7 (up to 13 %), and 9 of the splits that it leaves out would have gained 2-13 %.
               Not below 24 tiles (1,000 tokens over themselves: 31 us whole, 31-34 split), and into no more parts
               than min(scratch, PARTIAL_BYTES) holds the partials of.
    With a window a row tile's keys are those that it sees, wherever they lie. Below 24 tiles, where the row tiles leave
               half the chip idle, they are split as well, into parts of 3 tiles and more, if the tiles saved take
               longer than the merge's launch and bytes (D 128, times with the launch, q and the store, ~8 us: 24 row tiles
               of 10 key tiles 27.1 us whole, 21.5 in four; 3 of 14 23.9, in five 16.1; 12 of 7 15.0, in two 17.0; 144 of 7
               22.4, 28.2)."""
    longest = max([n for _, n, _ in spans])
    if window:
        longest = min(longest, window_tiles(window, sinks, 128, group) * KEYS)
    nt = -(-longest // KEYS)
    if nt < 24:
        if window:
            tasks = row_tiles(spans, group, 4) * hkv
            if 0 < 2 * tasks <= SLOTS[D]:
                chunk = max(3, -(-nt // (SLOTS[D] // tasks)))
                row = total_q * hkv * group * (D + 2) * 4
                cost = MERGE_US + -(-nt // chunk) * row * 2 / 2.5e6
                if (nt - chunk) * ALONE_US[D] > cost and -(-nt // chunk) * row <= min(scratch, PARTIAL_BYTES):
                    return 4, chunk
        return 4, 0
    if D <= 128 and longest >= 16384:
        wide = sum(c * (-(-t * group // 256)) for t, _, c in spans) * hkv              # row tiles of 8 waves
        if wide >= CUS and wide >= 0.8 * CUS * -(-wide // CUS):
            return 8, 0
    tasks = units = 0
    for t, n, c in spans:
        tiles = -(-t * group // 128) * c
        tasks += tiles
        keys = n - t // 2 if causal else n                                # (causal: the mean over the rows, N >= T)
        units += tiles * -(-(min(keys, longest) if window else keys) // KEYS)
    tasks, units = tasks * hkv, units * hkv
    if not tasks:
        return 4, 0
    slots = SLOTS[D]
    if 2 * tasks <= slots:
        chunk = -(-nt // (slots // tasks))
    else:
        chunk = -(-max(2 * units // slots, nt) // 2)
    row = total_q * hkv * group * (D + 2) * 4
    parts = min(scratch, PARTIAL_BYTES) // row                          # at most, in the scratch
    if parts < 2:
        return 4, 0
    chunk = max(chunk, 12, -(-nt // parts))
    gain = (0.7 if D == 256 else 0.5) * (nt - units / slots) * TILE_US[D]
    if chunk >= nt or gain <= -(-nt // chunk) * row * 2 / 2.5e6:
        return 4, 0
    return 4, chunk


@lru_cache(512)
def _window_plan(q_shape: tuple, k_shape: tuple, spans: tuple | None, scratch: int, window: int, sinks: int) -> tuple | None:
    """How a windowed call of these shapes runs: (n_q, n_k, waves, chunk, partial rows, row tiles of ragged rows, sequences); None where
    the kernel does not take them, or every query sees all. A step's layers ask for the same."""
    D, Hq, Hk = q_shape[-1], q_shape[-2], k_shape[-2]
    if (D not in SLOTS or k_shape[-1] != D or not Hk or Hq % Hk or 0 in q_shape or 0 in k_shape or len(k_shape) != len(q_shape)
            or len(q_shape) != (4 if spans is None else 3)):
        return None
    if spans is None:
        seqs, total = ((q_shape[1], k_shape[1], q_shape[0]),), q_shape[0] * q_shape[1]
        if k_shape[0] != q_shape[0]:
            return None
    else:
        seqs, total = tuple((t, n, 1) for t, n in spans), q_shape[0]
        if sum(t for t, _ in spans) != total or sum(n for _, n in spans) != k_shape[0]:
            return None
    n_q, n_k = max(s[0] for s in seqs), max(s[1] for s in seqs)
    group = Hq // Hk
    if any(s[0] < 0 or s[1] < s[0] for s in seqs) or n_q * group > 1 << 22 or n_k > 1 << 30 or window >= n_k:
        return None
    waves, chunk = plan(seqs, group, Hk, D, total, True, scratch, window, sinks)
    tiles = min(-(-n_k // KEYS), window_tiles(window, sinks, 32 * waves, group))
    rows = -(-tiles // chunk) * total * Hq if chunk else 0
    return n_q, n_k, waves, chunk, rows, 0 if spans is None else row_tiles(seqs, group, waves), q_shape[0] if spans is None else len(spans)


def window_native(q, k, v, scale, cu, spans, out, window, sinks, scratch: int = PARTIAL_BYTES):
    """A windowed call in native code (csrc/kush_stepcall.cpp, which checks the tensors), or None: not taken, nothing was
    launched."""
    m = _lib.native()
    if m is None or not q.is_cuda or not _plain(q, k, v) or (spans is None) != (cu is None):
        return None
    seqs = None if spans is None else tuple((int(t), int(n)) for t, n in spans)
    p = _window_plan(q.shape, k.shape, seqs, scratch, window, sinks)
    if p is None:
        return None
    return m.attend(q, k, v, out, *(cu or (None, None)), scale, window, sinks, *p, torch._C._cuda_getCurrentRawStream(q.get_device()))


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool, scale: float, lse: bool = False,
           cu: tuple | None = None, spans=None, out: torch.Tensor | None = None, scratch: int = PARTIAL_BYTES,
           window: int = 0, sinks: int = 0):
    """Attention of inputs that takes() accepts: out in q's shape and type (the given one, its rows 16-byte
    aligned, or a new one), or with lse the pair (out fp32, lse fp32 [.., Hq]). cu = (cu_q, cu_k, max_q, max_k)
    and spans = [(T, N)] for packed rows: the offsets as int32 device tensors, the lengths on the host. scratch: the
    bytes that partials of split keys may take. window (causal calls): of the keys up to its own a query sees the last
    `window` and the first `sinks` (0: all of them)."""
    D, Hq, Hk = q.shape[-1], q.shape[-2], k.shape[-2]
    group = Hq // Hk
    if cu is None:
        seqs, n_q, n_k, total = q.shape[0], q.shape[1], k.shape[1], q.shape[0] * q.shape[1]
        cq = ck = None
        window = 0 if window >= n_k else window
        waves, chunk = plan(((n_q, n_k, seqs),), group, Hk, D, total, causal, scratch, window, sinks)
    else:
        cq, ck, n_q, n_k = cu[0].data_ptr(), cu[1].data_ptr(), cu[2], cu[3]
        seqs, total = len(spans), q.shape[0]
        window = 0 if window >= n_k else window
        waves, chunk = plan([(t, n, 1) for t, n in spans], group, Hk, D, total, causal, scratch, window, sinks)
    dev = q.device
    if out is None:
        out = torch.empty(q.shape, dtype=torch.float32 if lse else q.dtype, device=dev)
    logs = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev) if lse else None
    ls = _row_strides(logs.unsqueeze(-1), 1) if lse else (0, 0, 0)
    strides = _Strides(*_row_strides(q, D), *_row_strides(k, D), *_row_strides(v, D), *_row_strides(out, D), *ls)
    tiles = -(-n_k // KEYS) if not window else min(-(-n_k // KEYS), window_tiles(window, sinks, 32 * waves, group))
    rows = -(-tiles // chunk) * total * Hq if chunk else 0                     # partial rows: every split's
    part = torch.empty(rows * (D + 2), dtype=torch.float32, device=dev) if chunk else None
    name = "kush_window_attend" if window else "kush_attend"
    limit = (window, sinks, row_tiles(spans, group, waves) if cu is not None else 0) if window else ()
    with torch.cuda.device(dev):
        rc = getattr(_lib.lib(), name)(
            D, 1 if q.dtype == torch.float16 else 2, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            logs.data_ptr() if lse else None, ctypes.addressof(strides), cq, ck, n_q, n_k, total, seqs, Hk, group, scale,
            *(() if window else (int(causal),)), int(lse), waves, chunk, part.data_ptr() if chunk else None,
            part.data_ptr() + rows * D * 4 if chunk else None, torch.cuda.current_stream(dev).cuda_stream, *limit)
    if rc:
        raise RuntimeError(f"{name} failed ({rc}): {(_lib.lib().kush_last_error() or b'').decode(errors='replace')}")
    return (out, logs) if lse else out
