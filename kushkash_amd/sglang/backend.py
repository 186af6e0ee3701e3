"""The "kushkash" SGLang attention backend on the gfx950 kernels: decode steps (capturable as HIP
graphs) and prefill / extend steps over the page records of ``KushPool``.
Reference semantics: kushkash/sglang/backend.py:146-404.

SGLang's bookkeeping, as the backend reads it:
  page of logical page p of a request   req_to_token[request slot, 32 p] // 32
  exact K tail slot                      the request-pool slot (stable while the request runs)
  seq_lens                               count this step's tokens (a decode token sits at seq_len - 1)

Decode step, per layer: one launch (``Ops.append_decode``) appends the step's token and attends over the
whole cache. Eager steps start the longest requests' workgroups first; captured steps use static
buffers sized by ``init_cuda_graph_state`` and a block table that spans the model's context.

Extend step, per layer: the attention reads the cache as it was before this step, then one
``Ops.write`` quantizes the new tokens. Requests are packed end to end in groups whose keys fit
KUSHKASH_PACK_MB (default 512 MiB of K + V): one unpack launch per group builds every request's
[history pages | exact tail | new tokens] keys, then a causal ragged attention runs over them with
the queries at the end of each request's keys. A request too long for one group, or every request
with KUSHKASH_PREFILL=loop, takes the history in blocks of pages instead (one unpack launch per block,
log-sum-exp merges), in bounded memory.

Rotation (KUSHKASH_ROTATE; auto: on for 4 bits): the records and tails hold Hadamard-rotated K and V.
The kernels rotate (canonical Walsh-Hadamard transform): the writes rotate new rows before they are
stored, the decode rotates q on load and its output back, and the unpack rotates history back, so
the prefill attention runs on the model's own q, k, v. No rotation product runs in torch.

Diagnostics and switches (kushkash_amd._serving): KUSHKASH_SYNC, KUSHKASH_CHECK, KUSHKASH_MEM_STATS and
KUSHKASH_UNPACK, with the reference's meanings.
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch
from sglang.srt.layers.attention.base_attn_backend import AttentionBackend

from .._ops import PAGE, Ops
from .._prefill import ExtendPlan, pack_budget, pack_plan, prefill_mode  # noqa: F401  (re-exported)
from .._rotation import rotation_enabled
from .._serving import Checker, MemStats, maybe_sync
from .._step import block_table
from .pool import KushPool


@dataclass
class _Step:
    """Metadata of one forward step, shared by its layers."""
    decode: bool
    block_table: torch.Tensor              # int32 [R, pages]
    seq_lens: torch.Tensor                 # int32 [R]
    slots: torch.Tensor                    # int32 [R]: request-pool slot = tail slot
    n_splits: int | None = None            # decode: chosen on the step's first layer unless set
    order: torch.Tensor | None = None      # decode: workgroup start order, longest request first
    extend: ExtendPlan | None = None       # extend: write jobs and attention groups


# layer attributes the backend cannot honour: (attribute, is set, message)
_LAYER_REFUSALS = (
    ("logit_cap", lambda x: bool(x) and x > 0, "logit soft-capping is not supported"),
    ("sliding_window_size", lambda x: x not in (None, -1), "sliding-window attention is not supported"),
    ("is_cross_attention", bool, "cross attention is not supported"),
)


def _rows(x: torch.Tensor, heads: int, dim: int) -> torch.Tensor:
    """[T, heads * dim] (row stride free) -> [T, heads, dim] rows with unit dim stride, head stride dim."""
    y = x.view(-1, heads, dim)
    return y if y.stride(2) == 1 and y.stride(1) == dim else y.contiguous()


class KushSGLangBackend(AttentionBackend):

    def __init__(self, runner):
        super().__init__()
        pool = runner.token_to_kv_pool
        if not isinstance(pool, KushPool):
            raise RuntimeError(f"kushkash: the attention backend runs on KushPool, but the server built a "
                               f"{type(pool).__name__} (hybrid, sliding-window and MLA models are not supported)")
        self.pool, self.rtp = pool, runner.req_to_token_pool
        self.device = pool.kush_records.device
        self.dtype = runner.model_config.dtype
        self.D, self.Hk, self.bits = pool.head_dim, pool.head_num, pool.kush_bits
        self.rot = rotation_enabled(self.bits)
        pool.ensure_tails(self.rtp.req_to_token.shape[0], self.dtype)
        self.max_pages = -(-self.rtp.req_to_token.shape[1] // PAGE)
        self.G = self._group_from_config(runner.model_config)
        self.prefill_mode = prefill_mode()
        self._ops: dict[int, Ops] = {}
        self.work = None
        self._graph = None
        self.forward_metadata = None
        self._mem = MemStats()

    def _group_from_config(self, model_config):
        """q heads per kv head from the model config, or None when it cannot be read (eager steps then
        take it from the layer; decode graphs refuse to start)."""
        try:
            from sglang.srt.runtime_context import get_parallel
            return model_config.get_num_attention_heads(get_parallel().attn_tp_size) // self.Hk
        except Exception:
            return None

    def _ops_for(self, G: int) -> Ops:
        ops = self._ops.get(G)
        if ops is None:
            ops = self._ops[G] = Ops(self.device, self.D, self.bits, G, self.dtype)
            # Ops.splits keeps requests x kv heads x splits within twice the CUs
            need = 2 * ops.sms * G * (self.D + 2)
            if need > (0 if self.work is None else self.work.numel()):
                self.work = torch.empty(need, dtype=torch.float32, device=self.device)
        return ops

    # ---------------------------------------------------------------- decode graphs
    def init_cuda_graph_state(self, max_bs: int, max_num_tokens: int):
        """Static metadata of captured decode steps; the kernels are loaded before any capture."""
        if self.G is None:
            raise RuntimeError("kushkash: the model config gave no query heads per KV head, which decode graphs "
                               "need before capture (run with --disable-cuda-graph)")
        self._graph = dict(block_table=torch.zeros((max_bs, self.max_pages), dtype=torch.int32, device=self.device),
                           seq_lens=torch.ones(max_bs, dtype=torch.int32, device=self.device),
                           slots=torch.zeros(max_bs, dtype=torch.int32, device=self.device))
        self._ops_for(self.G)

    def get_cuda_graph_seq_len_fill_value(self):
        # padded rows of a replay get request slot 0, which SGLang never hands out: its req_to_token row
        # stays 0 (page 0, the padding page) and its tail slot is 0, so padding touches no live data
        return 1

    def init_forward_metadata_out_graph(self, forward_batch, in_capture: bool = False):
        """Metadata of a captured decode step, for its capture and every replay: device work into the
        static buffers only (no host reads), so the step's preparation can be captured too."""
        fb = forward_batch
        if not fb.forward_mode.is_decode():
            raise NotImplementedError(f"kushkash: graphs are supported for decode steps only, got {fb.forward_mode}")
        if self._graph is None:
            raise RuntimeError("kushkash: decode graphs need init_cuda_graph_state first")
        req = fb.req_pool_indices
        R = req.shape[0]
        g = self._graph
        bt, sl, slots = g["block_table"][:R], g["seq_lens"][:R], g["slots"][:R]
        block_table(self.rtp.req_to_token, req.contiguous(), fb.seq_lens.contiguous(), self.max_pages, out=(bt, sl, slots))
        ops = self._ops_for(self.G)
        self.forward_metadata = _Step(True, bt, sl, slots, n_splits=ops.splits(R, self.Hk, self.max_pages))

    def init_forward_metadata_in_graph(self, forward_batch):
        pass

    # ---------------------------------------------------------------- eager metadata
    def init_forward_metadata(self, forward_batch):
        fb = forward_batch
        mode = fb.forward_mode
        if mode.is_idle():
            self.forward_metadata = None
            return
        if mode.is_target_verify() or mode.is_draft_extend_v2():
            raise NotImplementedError("kushkash: speculative decoding (target verify, draft extend) is not supported")
        req = fb.req_pool_indices
        if req.numel() == 0:
            self.forward_metadata = None
            return
        lens = (fb.seq_lens_cpu if fb.seq_lens_cpu is not None else fb.seq_lens.cpu()).numpy().astype(np.int64)
        pages = max(1, -(-int(lens.max()) // PAGE))
        step = _Step(mode.is_decode(), *block_table(self.rtp.req_to_token, req.contiguous(), fb.seq_lens.contiguous(), pages))
        if step.decode:
            if len(lens) > 1 and lens.min() != lens.max():
                order = np.argsort(-lens, kind="stable").astype(np.int32)
                step.order = torch.from_numpy(order).to(self.device)
        else:
            slots = getattr(fb, "req_pool_indices_cpu", None)
            slots = (slots if slots is not None else req.cpu()).numpy().astype(np.int64)
            step.extend = ExtendPlan.build(list(fb.extend_seq_lens_cpu), list(fb.extend_prefix_lens_cpu), slots,
                                           step.block_table,
                                           kv_heads=self.Hk, head_dim=self.D, dtype=self.dtype,
                                           packed=self.prefill_mode == "packed")
        self.forward_metadata = step

    # ---------------------------------------------------------------- forward
    def _check_layer(self, layer, kwargs):
        """Attention modifiers (ALiBi slopes, sinks, masks, ...) arrive as extra arguments or layer
        attributes; ignoring one would be silently wrong, so each one that is set is refused."""
        extra = sorted(name for name, value in kwargs.items() if value is not None and value is not False)
        if extra:
            raise NotImplementedError(f"kushkash: unsupported attention argument(s) {extra}: ALiBi, attention sinks "
                                      "and custom masks are not supported")
        for attr, is_set, message in _LAYER_REFUSALS:
            if is_set(getattr(layer, attr, None)):
                raise NotImplementedError(f"kushkash: {message}")

    def _layer_state(self, layer):
        Hq, Hk, D = layer.tp_q_head_num, layer.tp_k_head_num, layer.qk_head_dim
        if Hk != self.Hk or D != self.D:
            raise ValueError(f"kushkash: layer {layer.layer_id} has {Hk} kv heads of {D}, the pool {self.Hk} of {self.D}")
        ops = self._ops_for(Hq // Hk)
        return Hq, ops, self.pool.records(layer.layer_id), self.pool.tail(layer.layer_id)

    def forward_decode(self, q, k, v, layer, forward_batch, save_kv_cache=True, **kwargs):
        self._check_layer(layer, kwargs)
        step = self.forward_metadata
        if step is None:                               # idle or empty batch
            return q.new_empty((q.shape[0], layer.tp_q_head_num * layer.qk_head_dim))
        Hq, ops, cache, tail = self._layer_state(layer)
        q3 = q.reshape(-1, Hq, self.D).contiguous()
        out = torch.empty_like(q3)
        if step.n_splits is None:
            step.n_splits = ops.splits(q3.shape[0], self.Hk, step.block_table.shape[1])
        args = (cache, step.block_table, step.seq_lens, step.slots, tail, float(layer.scaling), step.n_splits,
                self.work)
        if save_kv_cache and k is not None:
            ops.append_decode(_rows(k, self.Hk, self.D), _rows(v, self.Hk, self.D), q3, out, *args, order=step.order,
                              rot=self.rot)
        else:
            ops.decode(q3, out, *args, order=step.order, rot=self.rot)
        if Checker.wanted(q3, layer.layer_id == 0):   # KUSHKASH_CHECK=<log>: layer 0 against torch
            R = q3.shape[0]
            Checker(self.D, ops.bits, float(layer.scaling), self.rot).log(
                out, q3, cache, step.block_table, tail, step.slots.cpu().tolist(), list(range(R + 1)),
                step.seq_lens.cpu().tolist(), R, {})
        maybe_sync(out)                                # KUSHKASH_SYNC=1
        return out.view(-1, Hq * self.D)

    def forward_extend(self, q, k, v, layer, forward_batch, save_kv_cache=True, **kwargs):
        self._check_layer(layer, kwargs)
        step = self.forward_metadata
        if step is None:
            return q.new_empty((q.shape[0], layer.tp_q_head_num * layer.qk_head_dim))
        Hq, ops, cache, tail = self._layer_state(layer)
        q3 = q.reshape(-1, Hq, self.D)
        k3, v3 = _rows(k, self.Hk, self.D), _rows(v, self.Hk, self.D)
        plan = step.extend
        first = layer.layer_id == 0
        check = Checker.wanted(q3, first)              # KUSHKASH_CHECK=<log>: layer 0 against torch
        if check:
            chk = Checker(self.D, ops.bits, float(layer.scaling), self.rot)
            slots = step.slots.cpu().tolist()
            refs = chk.prefill_refs(q3, k3, v3, cache, step.block_table, tail, slots, plan.q_start_host,
                                    plan.history_host, range(len(plan.history_host)))
        if first and any(g.packed and g.has_history for g in plan.groups):
            self._mem.tick(q3.device)                  # KUSHKASH_MEM_STATS=N
        out = plan.attend(ops, q3, k3, v3, cache, tail, step.block_table, step.slots, float(layer.scaling), self.rot)
        if save_kv_cache:
            plan.write(ops, k3, v3, step.seq_lens, step.slots, cache, step.block_table, tail, self.rot)
        if check:
            chk.log(out, q3, cache, step.block_table, tail, slots, plan.q_start_host, step.seq_lens.cpu().tolist(), 0,
                    refs)
        maybe_sync(out)                                # KUSHKASH_SYNC=1
        return out.view(-1, Hq * self.D)
