"""vLLM attention backend over the B200 split-KV decode kernels.

The reference runs attention inside its DecodeLayer megakernel and reads vLLM's paged
metadata through ``get_attention_context`` (integration/model.py:49, 64-69): the block
table, the slot mapping and the sequence lengths.  This backend supplies the same
metadata to the sm_100a kernels:

* KV cache: ``[2, num_blocks, num_kv_heads, block_size, head_size]`` bf16, i.e. for K
  and for V one (block, kv head) page of 128 tokens x 128 dims contiguous, the layout
  ``spark_attn_splitkv`` streams;
* decode (one query token per request): ``spark_kv_store`` writes this step's k / v at
  the slot mapping, then split-KV attention with the fused log-sum-exp combine per
  request (``spark_attn_decode``); uniform single-token decode batches are CUDA-graph
  capturable;
* head_size 256 and sliding-window layers (the reference's Spark model,
  plugin/spark2_5.py:140-241): decode runs the persistent step kernel's attention stage
  as a one-stage program (``spark_step_run``, its Spark instantiation: 16 lanes per
  token, the window's positions only).  A sliding window of W attends to W + 1
  positions, the current one included, as the reference's kernel does (it masks below
  len - 513 for its 512-window layers, kernels/attention.py:124-127);
* prefill (query length > 1) is not on the decode hot path: causal attention in torch
  over the request's gathered pages, on the GPU;
* with ``SPARK_B200_PAGED_ATTENTION=1`` every step that is not all single tokens (prompts,
  chunks, mixed batches) runs the paged attention kernel instead (``ops.attn_prompt_out``:
  one launch for all requests, reading the pages in place, no host copy of the lengths), and
  the backend asks vLLM for cascade attention, so that decode batches with a common prefix
  read it once (``ops.attn_shared_prefix_out``).  Off by default: its probabilities are
  rounded to bf16 where the torch path's are fp32, so its outputs differ by up to 2^-8 of
  sum p |v| (several bf16 steps where the sum cancels).  What a step's kernels report is
  raised when a later step is built (``raise_on_error`` waits for it).
"""
from __future__ import annotations

import math
import os
import threading
import weakref
from dataclasses import dataclass, field
from typing import ClassVar

import ctypes

import torch
from vllm.config import get_current_vllm_config_or_none
from vllm.v1.attention.backend import (AttentionBackend, AttentionCGSupport, AttentionImpl, AttentionMetadataBuilder,
                                       AttentionType, CommonAttentionMetadata)

from .. import ops

BLOCK_SIZE = 128
HEAD_SIZE = 128
PAGED_ENV = "SPARK_B200_PAGED_ATTENTION"
HEAD_SIZES = (128, 256)  # 256: the persistent kernel's attention stage (the Spark model)


def paged_attention() -> bool:
    return os.environ.get(PAGED_ENV, "").strip().lower() in ("1", "true", "yes", "on")


def choose_splits(max_model_len: int) -> int:
    """Splits of at most 128 tokens (one cache page), between 16 and 256 (the fused
    combine's limit)."""
    return min(256, max(16, -(-max_model_len // BLOCK_SIZE)))


def split_tokens(max_model_len: int, splits: int) -> int:
    return (math.ceil(max_model_len / splits) + 15) // 16 * 16


@dataclass
class SparkAttentionMetadata:
    num_actual_tokens: int
    num_reqs: int
    max_query_len: int
    max_seq_len: int
    query_start_loc: torch.Tensor  # int32 [num_reqs + 1]
    query_start_loc_cpu: torch.Tensor
    seq_lens: torch.Tensor  # int32 [num_reqs] (device)
    block_table: torch.Tensor  # int32 [num_reqs, max_blocks]
    slot_mapping: torch.Tensor  # int64 [num_tokens]
    splits: int
    max_split_tokens: int
    prefix_len: torch.Tensor | None = None  # int32 [1]: positions all requests share (cascade)
    plans: dict = field(default_factory=dict)  # this step's attention work lists, per head layout and window
    layers_left: int = 0  # paged attention calls until the step's last (0: not known)

    @property
    def is_decode(self) -> bool:
        return self.max_query_len == 1


def _settle(device) -> None:
    """What was just zeroed on the current stream may be another stream's from now on."""
    if torch.device(device).type == "cuda" and not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream(device).synchronize()


class StepStatus:
    """The status word of a device's paged steps (ERR_* bits of plans and attention calls) and its
    way to the host: copied to pinned memory behind a step's last layer, looked at when a later
    step is built, so that nothing waits.  A copy that is under way is looked at before the next
    one is made, whose event would take its place."""

    def __init__(self, device):
        self.word = torch.zeros(1, dtype=torch.int32, device=device)
        cuda = self.word.is_cuda
        self._host = torch.zeros(1, dtype=torch.int32, pin_memory=cuda)
        self._event = torch.cuda.Event() if cuda else None
        self._stream = None
        self._used = self._posted = False
        _settle(device)

    def used(self) -> None:
        """A call that may set bits was queued on the current stream."""
        self._used = True
        if self._event is not None:
            self._stream = torch.cuda.current_stream(self.word.device)

    def post(self) -> None:
        if not self._used or self._posted:
            return
        if self._event is None:
            self._host.copy_(self.word)
        else:
            with torch.cuda.stream(self._stream):
                if torch.cuda.is_current_stream_capturing():
                    return
                self._host.copy_(self.word, non_blocking=True)
                self._event.record()
        self._used, self._posted = False, True

    def check(self, wait: bool = False) -> None:
        """Raise if a copy that has arrived (``wait``: the one under way, too) holds bits."""
        if not self._posted:
            return
        if self._event is not None:
            if wait:
                self._event.synchronize()
            elif not self._event.query():
                return
        self._posted = False
        bits = int(self._host)
        if bits:
            if self._stream is not None:
                with torch.cuda.stream(self._stream):
                    self.word.zero_()
            else:
                self.word.zero_()
            raise RuntimeError(f"paged attention: a step reported status {bits} (spark_b200.ops.ERR_* bits): "
                               "its outputs are not valid")


class PlanPool:
    """Attention plans (``ops.AttnPlan``) kept from step to step.

    A plan holds one work list at a time, and every layer of a step reads it.  So metadata
    objects that are alive together (micro-batches whose layers take turns, cache groups of
    one layout) get a plan each: one is free again when the metadata object that took it is
    gone.  Work that is still queued then stays in front of the next list's on the plan's
    stream; a plan that was used is not handed to another stream."""

    def __init__(self):
        self._plans: dict = {}  # (head layout, window, device) -> [[plan, its metadata, its stream]]
        self._status: dict = {}
        self._lock = threading.RLock()  # (micro-batches may run in threads of their own)

    def status(self, device) -> StepStatus:
        st = self._status.get(str(device))
        if st is None:
            with self._lock:
                st = self._status.get(str(device)) or self._status.setdefault(str(device), StepStatus(device))
        return st

    def check(self, wait: bool = False) -> None:
        """Raise what earlier steps reported, and send for what has been used since."""
        for st in self._status.values():
            st.check(wait)
            st.post()
            if wait:
                st.check(wait)

    @staticmethod
    def _stream(device):
        return torch.cuda.current_stream(device) if torch.device(device).type == "cuda" else None

    def _make(self, layout, device, tokens: int, reqs: int):
        room = lambda n: 1 << max(n - 1, 63).bit_length()  # noqa: E731
        plan = ops.AttnPlan(room(tokens), room(reqs), *layout[:3], device, layout[3])
        plan.status = self.status(device)
        plan.error = plan.status.word
        return plan

    def reserve(self, layout, device, tokens: int, reqs: int) -> None:
        """Have a plan of this layout before the first step, bound to no stream yet (vLLM's
        profiling run counts the memory that is taken then)."""
        with self._lock:
            entries = self._plans.setdefault((*layout, str(device)), [])
            if not entries:
                plan = self._make(layout, device, tokens, reqs)
                _settle(device)
                entries.append([plan, lambda: None, None])

    def take(self, layout, device, tokens: int, reqs: int, owner):
        """A plan for up to ``tokens`` tokens and ``reqs`` requests that ``owner`` alone uses."""
        with self._lock:
            entries = self._plans.setdefault((*layout, str(device)), [])
            stream = self._stream(device)
            free = [e for e in entries if e[1]() is None and e[2] in (None, stream)]
            for e in free:
                if e[0].max_tokens >= tokens and e[0].max_reqs >= reqs:
                    if e[2] is None and stream is not None:  # (its memory may be another stream's)
                        for t in (e[0].buf, e[0].part_o, e[0].part_ml):
                            t.record_stream(stream)
                    e[1], e[2] = weakref.ref(owner), stream
                    return e[0]
            if free:  # too small: a larger one in its place
                tokens, reqs = max(tokens, free[0][0].max_tokens), max(reqs, free[0][0].max_reqs)
                entries.remove(free[0])
            plan = self._make(layout, device, tokens, reqs)
            entries.append([plan, weakref.ref(owner), stream])
            return plan


_pool = PlanPool()


def raise_on_error() -> None:
    """Wait for the paged steps that are queued and raise if one reported an error.  (Without a
    call, a step's error is raised when a later step is built.)"""
    _pool.check(wait=True)


class SparkAttentionMetadataBuilder(AttentionMetadataBuilder[SparkAttentionMetadata]):
    _cudagraph_support: ClassVar[AttentionCGSupport] = AttentionCGSupport.UNIFORM_SINGLE_TOKEN_DECODE

    def __init__(self, kv_cache_spec, layer_names, vllm_config, device):
        super().__init__(kv_cache_spec, layer_names, vllm_config, device)
        max_len = vllm_config.model_config.max_model_len if vllm_config is not None else 4096
        self.splits = choose_splits(max_len)
        self.max_split_tokens = split_tokens(max_len, self.splits)

    def use_cascade_attention(self, common_prefix_len: int, query_lens, num_query_heads: int, num_kv_heads: int,
                              use_alibi: bool, use_sliding_window: bool, use_local_attention: bool, num_sms: int,
                              dcp_world_size: int) -> bool:
        """Single-token decode of two requests or more behind at least a page in common (the
        per-request path launches once per request and reads the prefix each time)."""
        return (paged_attention() and common_prefix_len >= BLOCK_SIZE and len(query_lens) > 1 and
                all(int(n) == 1 for n in query_lens) and not (use_alibi or use_sliding_window or use_local_attention)
                and dcp_world_size == 1)

    def build(self, common_prefix_len: int, common_attn_metadata: CommonAttentionMetadata,
              fast_build: bool = False) -> SparkAttentionMetadata:
        cm = common_attn_metadata
        _pool.check()
        prefix = None
        if common_prefix_len > 0:
            prefix = torch.full((1,), common_prefix_len, dtype=torch.int32, device=cm.seq_lens.device)
        return SparkAttentionMetadata(
            prefix_len=prefix, layers_left=len(getattr(self, "layer_names", ())),
            num_actual_tokens=cm.num_actual_tokens, num_reqs=cm.num_reqs, max_query_len=cm.max_query_len,
            max_seq_len=cm.max_seq_len, query_start_loc=cm.query_start_loc, query_start_loc_cpu=cm.query_start_loc_cpu,
            seq_lens=cm.seq_lens, block_table=cm.block_table_tensor, slot_mapping=cm.slot_mapping,
            splits=self.splits, max_split_tokens=self.max_split_tokens)


class SparkAttentionImpl(AttentionImpl[SparkAttentionMetadata]):
    def __init__(self, num_heads: int, head_size: int, scale: float, num_kv_heads: int | None = None,
                 alibi_slopes: list[float] | None = None, sliding_window: int | None = None,
                 kv_cache_dtype: str = "auto", logits_soft_cap: float | None = None,
                 attn_type: str = AttentionType.DECODER, kv_sharing_target_layer_name: str | None = None) -> None:
        if head_size not in HEAD_SIZES:
            raise ValueError(f"SparkAttentionBackend supports head_size {HEAD_SIZES}, got {head_size}")
        if alibi_slopes is not None or logits_soft_cap:
            raise NotImplementedError("SparkAttentionBackend: alibi / soft cap are not supported")
        if sliding_window is not None and head_size != 256:
            raise NotImplementedError("SparkAttentionBackend: sliding windows with head_size 256 only")
        if head_size == 256 and num_heads != 4 * (num_kv_heads or num_heads):
            raise NotImplementedError("SparkAttentionBackend: head_size 256 needs 4 query heads per kv head")
        if attn_type != AttentionType.DECODER:
            raise NotImplementedError("SparkAttentionBackend: decoder self-attention only")
        if kv_cache_dtype not in ("auto", "bfloat16"):
            raise NotImplementedError("SparkAttentionBackend: bf16 KV cache only")
        self.num_heads = num_heads
        self.head_size = head_size
        self.num_kv_heads = num_kv_heads or num_heads
        self.scale = float(scale)
        self.kv_cache_dtype = kv_cache_dtype
        self.kv_sharing_target_layer_name = kv_sharing_target_layer_name
        # positions attended by a sliding layer (the reference's 512-window layers: 513)
        self.window = sliding_window + 1 if sliding_window is not None else 0
        self._ws: dict = {}
        self._step = None
        self._paged = paged_attention()
        self._error: dict = {}
        self._layout = (num_heads, self.num_kv_heads, head_size, self.window)
        config = get_current_vllm_config_or_none()
        self._max_reqs = config.scheduler_config.max_num_seqs if config is not None else 1

    def _workspace(self, splits: int, device) -> tuple:
        key = (splits, device)
        ws = self._ws.get(key)
        if ws is None:
            nq, d = self.num_heads, self.head_size
            ws = (torch.empty((splits, nq, d), dtype=torch.float32, device=device),
                  torch.empty((splits, nq), dtype=torch.float32, device=device),
                  torch.zeros(self.num_kv_heads, dtype=torch.int32, device=device),  # left zero by the kernel
                  torch.zeros(1, dtype=torch.int32, device=device))
            self._ws[key] = ws
        return ws

    def forward(self, layer, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor,
                attn_metadata: SparkAttentionMetadata, output: torch.Tensor, output_scale: torch.Tensor | None = None,
                output_block_scale: torch.Tensor | None = None) -> torch.Tensor:
        if attn_metadata is None:  # profiling run
            if self._paged and not (query.is_cuda and torch.cuda.is_current_stream_capturing()):
                _pool.reserve(self._layout, query.device, query.shape[0], self._max_reqs)
            return output.fill_(0)
        md = attn_metadata
        nq, nkv, d = self.num_heads, self.num_kv_heads, self.head_size
        t = md.num_actual_tokens
        q = query[:t].view(t, nq, d)
        k_cache, v_cache = kv_cache[0], kv_cache[1]
        if self.kv_sharing_target_layer_name is None and key is not None:
            ops.kv_store_(key[:t].view(t, nkv, d), value[:t].view(t, nkv, d), md.slot_mapping[:t], k_cache, v_cache)
        out = output[:t].view(t, nq, d)
        if self._paged and (not md.is_decode or (md.prefix_len is not None and not self.window)):
            return self._paged_attention(q, k_cache, v_cache, md, out, output)
        if md.is_decode and (d != HEAD_SIZE or self.window):
            return self._decode_step(q, key, value, k_cache, v_cache, md, out, output)
        if md.is_decode:
            part_o, part_lse, counters, err = self._workspace(md.splits, query.device)
            for r in range(md.num_reqs):  # one query token per request
                ops.attn_decode_out(q[r], k_cache, v_cache, md.block_table[r], md.splits, md.max_split_tokens,
                                    self.scale, part_o, part_lse, counters, out[r], seq_len=md.seq_lens[r:r + 1],
                                    error=err)
            return output
        return self._prefill(q, k_cache, v_cache, md, out, output)

    def _plan(self, md, device):
        """This step's work list: made by the first layer of a head layout and window, used
        by the others."""
        key = self._layout
        plan = md.plans.get(key)
        if plan is None:
            reqs = md.num_reqs
            plan = _pool.take(key, device, max(md.num_actual_tokens, reqs), reqs, md)
            if md.is_decode and md.prefix_len is not None and not self.window:
                plan.update_prefix(md.seq_lens[:reqs], md.prefix_len)
            else:
                plan.update(md.query_start_loc[:reqs + 1], md.seq_lens[:reqs])
            md.plans[key] = plan
        return plan

    def _paged_attention(self, q, k_cache, v_cache, md, out, output):
        plan = self._plan(md, q.device)
        status = plan.status
        self._error[q.device] = status.word
        status.used()
        attend = ops.attn_prompt_out if plan.kind == "prompt" else ops.attn_shared_prefix_out
        attend(q, k_cache, v_cache, md.block_table, plan, self.scale, out, status.word)
        md.layers_left -= 1
        if md.layers_left == 0:
            status.post()
        return output

    def _step_state(self, md, device):
        """Persistent buffers of the one-stage step-kernel program (fixed pointers, so a
        captured decode graph replays them): partials, head counters, launch counters,
        this step's k / v per request, positions, the error word."""
        from .. import step as S
        if self._step is None:
            nq, nkv, d = self.num_heads, self.num_kv_heads, self.head_size
            ncta = S.num_ctas()
            max_len = md.splits * md.max_split_tokens  # the builder's bound on the model length
            splits = S.splits_for(nkv, ncta, max_len, d)
            z = lambda *sh, dt=torch.float32: torch.zeros(sh, dtype=dt, device=device)  # noqa: E731
            self._step = {"splits": splits, "T": S.max_split_tokens(max_len, splits), "part_o": z(splits, nq, d),
                          "part_lse": z(splits, nq), "head_ctr": z(nkv, dt=torch.int32),
                          "counters": z(4, dt=torch.int32), "error": z(1, dt=torch.int32), "kv_new": {}, "pos": {}}
        return self._step

    def _decode_step(self, q, key, value, k_cache, v_cache, md, out, output):
        from .. import step as S
        from .._lib import SparkStage, call
        st_ = self._step_state(md, q.device)
        nq, nkv, d, R = self.num_heads, self.num_kv_heads, self.head_size, md.num_reqs
        kvn = st_["kv_new"].get(R)
        if kvn is None:
            kvn = st_["kv_new"][R] = torch.zeros((R, 2, nkv, d), dtype=torch.bfloat16, device=q.device)
            st_["pos"][R] = torch.zeros(R, dtype=torch.int64, device=q.device)
        pos = st_["pos"][R]
        kvn[:, 0].copy_(key[:R].view(R, nkv, d))
        kvn[:, 1].copy_(value[:R].view(R, nkv, d))
        pos.copy_(md.seq_lens[:R])
        pos.sub_(1)
        io = S.SparkStepIO()
        io.counters, io.error, io.tp_size = ctypes.c_void_p(st_["counters"].data_ptr()), \
            ctypes.c_void_p(st_["error"].data_ptr()), 1
        for r in range(R):  # one query token per request
            stg = SparkStage()
            stg.kind, stg.wait = S.STAGE_ATTN, -1
            stg.nq, stg.nkv, stg.head_dim, stg.block_size = nq, nkv, d, k_cache.shape[2]
            stg.splits, stg.max_split_tokens, stg.scale, stg.window = st_["splits"], st_["T"], self.scale, self.window
            for name, tns in (("q", q[r]), ("k_cache", k_cache), ("v_cache", v_cache), ("kv_new", kvn[r]),
                              ("block_table", md.block_table[r]), ("pos", pos[r:r + 1]),
                              ("part_o", st_["part_o"]), ("part_lse", st_["part_lse"]),
                              ("head_counters", st_["head_ctr"]), ("attn_out", out[r])):
                setattr(stg, name, ctypes.c_void_p(tns.data_ptr()))
            call("spark_step_run", ctypes.byref(stg), None, 1, ctypes.byref(io), S._stream())
        return output

    def _prefill(self, q, k_cache, v_cache, md, out, output):
        qsl = md.query_start_loc_cpu.tolist()
        seq = md.seq_lens.tolist()
        group = self.num_heads // self.num_kv_heads
        bs = k_cache.shape[2]
        for r in range(md.num_reqs):
            q0, q1, n = qsl[r], qsl[r + 1], seq[r]
            if q1 <= q0:
                continue
            nblk = -(-n // bs)
            pages = md.block_table[r, :nblk].long()
            kr = k_cache[pages].permute(1, 0, 2, 3).reshape(self.num_kv_heads, nblk * bs, -1)[:, :n]
            vr = v_cache[pages].permute(1, 0, 2, 3).reshape(self.num_kv_heads, nblk * bs, -1)[:, :n]
            kr = kr.repeat_interleave(group, dim=0)
            vr = vr.repeat_interleave(group, dim=0)
            qr = q[q0:q1].transpose(0, 1)  # [nq, lq, d]
            lq = q1 - q0
            # query i sits at absolute position n - lq + i and sees keys 0 .. n - lq + i
            qpos = (n - lq + torch.arange(lq, device=q.device))[:, None]
            kpos = torch.arange(n, device=q.device)[None, :]
            mask = kpos <= qpos
            if self.window:  # (sliding layers: the last `window` positions)
                mask &= kpos > qpos - self.window
            o = torch.nn.functional.scaled_dot_product_attention(qr.float(), kr.float(), vr.float(), attn_mask=mask,
                                                                 scale=self.scale)
            out[q0:q1] = o.transpose(0, 1).to(out.dtype)
        return output


class SparkAttentionBackend(AttentionBackend):
    supported_dtypes: ClassVar[list[torch.dtype]] = [torch.bfloat16]
    supported_kv_cache_dtypes: ClassVar[list] = ["auto", "bfloat16"]
    forward_includes_kv_cache_update: bool = True

    @staticmethod
    def get_name() -> str:
        return "CUSTOM"

    @staticmethod
    def get_impl_cls():
        return SparkAttentionImpl

    @staticmethod
    def get_builder_cls():
        return SparkAttentionMetadataBuilder

    @staticmethod
    def get_kv_cache_shape(num_blocks: int, block_size: int, num_kv_heads: int, head_size: int,
                           cache_dtype_str: str = "auto") -> tuple[int, ...]:
        return (2, num_blocks, num_kv_heads, block_size, head_size)

    @staticmethod
    def get_supported_kernel_block_sizes() -> list[int]:
        return [BLOCK_SIZE]

    @classmethod
    def get_supported_head_sizes(cls) -> list[int]:
        return list(HEAD_SIZES)
