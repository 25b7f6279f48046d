"""Torch-facing operators over the C ABI, plus ``torch.ops.spark_b200.*`` registrations.

Two layers:

* ``*_out`` functions take caller-owned output tensors, allocate nothing and
  launch on the current CUDA stream -- this is what the decode engine captures
  into a CUDA graph.
* ``torch.ops.spark_b200.<name>`` custom ops (``torch.library.custom_op``) that
  allocate their outputs; they are what the vLLM quantized-linear method and
  attention backend call.  Each has a fake (meta) implementation so that
  torch.compile can trace through it.

Argument checks mirror the reference's native op (native/head/extension.cpp:8-10):
device, dtype, layout and size are validated before the launch, and a bad call
raises instead of reaching the kernel.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import call, lib

BF16 = torch.bfloat16


def _p(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream() -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _cuda(t: torch.Tensor, name: str, dtype: torch.dtype | None = None) -> None:
    _check(t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.is_contiguous(), f"{name} must be contiguous")
    if dtype is not None:
        _check(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")


def _q4(qs: torch.Tensor, d: torch.Tensor) -> tuple[int, int]:
    _cuda(qs, "qs", torch.uint8)
    _cuda(d, "d")
    _check(d.dtype in (torch.float16, torch.uint16, torch.int16), "d must hold fp16 scales")
    _check(qs.dim() == 2 and d.dim() == 2, "qs / d must be 2-D")
    n, k = qs.shape[0], qs.shape[1] * 2
    _check(d.shape == (n, k // 32), f"d must be [{n}, {k // 32}], got {tuple(d.shape)}")
    return n, k


# ---------------------------------------------------------------- Q4_0 format
def q4_quantize(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 [rows, k] on the GPU -> (qs uint8 [rows, k/2], d fp16 [rows, k/32]); gguf Q4_0."""
    _cuda(w, "w", torch.float32)
    rows, k = w.shape
    qs = torch.empty((rows, k // 2), dtype=torch.uint8, device=w.device)
    d = torch.empty((rows, k // 32), dtype=torch.float16, device=w.device)
    call("spark_q4_quantize", _p(w), rows, k, _p(qs), _p(d), _stream())
    return qs, d


def q4_split_gguf(blocks: torch.Tensor, rows: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    _cuda(blocks, "blocks", torch.uint8)
    _check(blocks.numel() == rows * (k // 32) * 18, "blocks size mismatch")
    qs = torch.empty((rows, k // 2), dtype=torch.uint8, device=blocks.device)
    d = torch.empty((rows, k // 32), dtype=torch.float16, device=blocks.device)
    call("spark_q4_split_gguf", _p(blocks), rows, k, _p(qs), _p(d), _stream())
    return qs, d


def q4_dequantize(qs: torch.Tensor, d: torch.Tensor) -> torch.Tensor:
    n, k = _q4(qs, d)
    w = torch.empty((n, k), dtype=BF16, device=qs.device)
    call("spark_q4_dequantize_bf16", _p(qs), _p(d), n, k, _p(w), _stream())
    return w


def q4_gemm(x: torch.Tensor, qs: torch.Tensor, d: torch.Tensor, error: torch.Tensor,
            wait_ns: int = -1) -> torch.Tensor:
    """Prefill GEMM on the tensor cores: x bf16 [T, K] times the Q4_0 weight [N, K]
    (dequantized in shared memory) -> bf16 [T, N].  K % 256 == 0.  ``error`` (int32 [1],
    required, on the device) becomes nonzero if a wait inside the kernel ran out, and y
    is then not valid: the caller owns the status word and must read it.  ``wait_ns``
    bounds each wait (-1: the kernel's 0.5 s; 0: give up at once, for tests)."""
    n, k = _q4(qs, d)
    _cuda(x, "x", BF16)
    _cuda(error, "error", torch.int32)
    _check(error.numel() >= 1, "error must hold one int32")
    x2 = x.reshape(-1, k)
    _check(x2.is_contiguous(), "x must be contiguous")
    t = x2.shape[0]
    y = torch.empty((t, n), dtype=BF16, device=x.device)
    call("spark_q4_gemm_tc", _p(x2), _p(qs), _p(d), _p(y), t, n, k, _p(error), int(wait_ns), _stream())
    return y


# ---------------------------------------------------------------- GEMV family
def q4_gemv_out(x: torch.Tensor, qs: torch.Tensor, d: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    n, k = _q4(qs, d)
    _cuda(x, "x", BF16)
    _cuda(y, "y", BF16)
    x2 = x.reshape(-1, k)
    batch = x2.shape[0]
    _check(1 <= batch <= 8, "batch must be in 1..8")
    _check(y.numel() == batch * n, "y has the wrong size")
    call("spark_q4_gemv", _p(x2), _p(qs), _p(d), _p(y), n, k, batch, _stream())
    return y


def q4_gemv(x: torch.Tensor, qs: torch.Tensor, d: torch.Tensor) -> torch.Tensor:
    n, k = _q4(qs, d)
    y = torch.empty((*x.shape[:-1], n), dtype=BF16, device=x.device)
    return q4_gemv_out(x, qs, d, y)


def rmsnorm_q4_gemv_out(a, b, gamma, eps, qs, d, y, res_out=None):
    n, k = _q4(qs, d)
    for t, nm in ((a, "a"), (gamma, "gamma"), (y, "y")):
        _cuda(t, nm, BF16)
    _check(a.numel() == k and gamma.numel() == k and y.numel() == n, "size mismatch")
    if b is not None:
        _cuda(b, "b", BF16)
    call("spark_rmsnorm_q4_gemv", _p(a), _p(b), _p(gamma), float(eps), _p(res_out), _p(qs), _p(d), _p(y), n, k,
         _stream())
    return y


def rmsnorm_gate_up_silu_out(a, b, gamma, eps, qs, d, mid, res_out=None):
    n, k = _q4(qs, d)
    for t, nm in ((a, "a"), (gamma, "gamma"), (mid, "mid")):
        _cuda(t, nm, BF16)
    _check(a.numel() == k and mid.numel() == n // 2, "size mismatch")
    call("spark_rmsnorm_gate_up_silu", _p(a), _p(b), _p(gamma), float(eps), _p(res_out), _p(qs), _p(d), _p(mid), n,
         k, _stream())
    return mid


def qkv_rope_kvstore_out(a, b, gamma, eps, qs, d, nq, nkv, head_dim, cos_sin, pos, block_table, slot_mapping,
                         block_size, k_cache, v_cache, q_out, res_out=None, embed=None, token=None):
    n, k = _q4(qs, d)
    _check(n == (nq + 2 * nkv) * head_dim, "qkv weight rows must be (nq + 2 nkv) * head_dim")
    _cuda(gamma, "gamma", BF16)
    _cuda(cos_sin, "cos_sin", BF16)
    _cuda(k_cache, "k_cache", BF16)
    _cuda(v_cache, "v_cache", BF16)
    _cuda(q_out, "q_out", BF16)
    _cuda(pos, "pos", torch.int64)
    call("spark_qkv_rope_kvstore", _p(a), _p(b), _p(embed), _p(token), _p(gamma), float(eps), _p(res_out), _p(qs),
         _p(d), k, nq, nkv, head_dim, _p(cos_sin), _p(pos), _p(block_table), _p(slot_mapping), block_size,
         _p(k_cache), _p(v_cache), _p(q_out), _stream())
    return q_out


def head_argmax_out(a, b, gamma, eps, qs, d, logits, key):
    n, k = _q4(qs, d)
    _cuda(logits, "logits", BF16)
    _check(key.dtype in (torch.int64, torch.uint64) and key.is_cuda, "key must be a CUDA int64 tensor")
    call("spark_rmsnorm_q4_head_argmax", _p(a), _p(b), _p(gamma), float(eps), _p(qs), _p(d), _p(logits), n, k,
         _p(key), _stream())
    return logits


def decode_finalize(key, token_out, token_log=None, step=None, pos=None):
    call("spark_decode_finalize", _p(key), _p(token_out), _p(token_log), _p(step), _p(pos), _stream())


# ---------------------------------------------------------------- attention
def attn_splitkv_out(q, k_cache, v_cache, block_table, splits, max_split_tokens, scale, part_o, part_lse,
                     pos=None, seq_len=None, error=None):
    _cuda(q, "q", BF16)
    nq, head_dim = q.shape[-2], q.shape[-1]
    _cuda(k_cache, "k_cache", BF16)
    _cuda(v_cache, "v_cache", BF16)
    _check(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "caches must be [blocks, nkv, block_size, D]")
    nkv, block_size = k_cache.shape[1], k_cache.shape[2]
    _check(k_cache.shape[3] == head_dim, "head_dim mismatch")
    _cuda(block_table, "block_table", torch.int32)
    _check(part_o.shape == (splits, nq, head_dim) and part_lse.shape == (splits, nq), "partials shape")
    _check((pos is None) != (seq_len is None), "give exactly one of pos / seq_len")
    if pos is not None:
        _cuda(pos, "pos", torch.int64)
    if seq_len is not None:
        _cuda(seq_len, "seq_len", torch.int32)
    call("spark_attn_splitkv", _p(q), _p(k_cache), _p(v_cache), _p(block_table), _p(pos), _p(seq_len), nq, nkv,
         head_dim, block_size, splits, max_split_tokens, float(scale), _p(part_o), _p(part_lse), _p(error), _stream())


def attn_decode_out(q, k_cache, v_cache, block_table, splits, max_split_tokens, scale, part_o, part_lse, counters,
                    out, pos=None, seq_len=None, error=None):
    """Split-KV attention with the fused LSE combine (counters: int32 [nkv], zero)."""
    _cuda(q, "q", BF16)
    nq, head_dim = q.shape[-2], q.shape[-1]
    _check(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "caches must be [blocks, nkv, block_size, D]")
    nkv, block_size = k_cache.shape[1], k_cache.shape[2]
    _cuda(counters, "counters", torch.int32)
    _cuda(out, "out", BF16)
    _check((pos is None) != (seq_len is None), "give exactly one of pos / seq_len")
    call("spark_attn_decode", _p(q), _p(k_cache), _p(v_cache), _p(block_table), _p(pos), _p(seq_len), nq, nkv,
         head_dim, block_size, splits, max_split_tokens, float(scale), _p(part_o), _p(part_lse), _p(counters),
         _p(out), _p(error), _stream())
    return out


def attn_combine_out(part_o, part_lse, out):
    splits, nq, head_dim = part_o.shape
    _cuda(part_o, "part_o", torch.float32)
    _cuda(part_lse, "part_lse", torch.float32)
    _cuda(out, "out", BF16)
    call("spark_attn_combine", _p(part_o), _p(part_lse), splits, nq, head_dim, _p(out), _stream())
    return out


# ---------------------------------------------------------------- elementwise
def add_rmsnorm_out(a, b, gamma, eps, y, res_out=None):
    _cuda(a, "a", BF16)
    _cuda(gamma, "gamma", BF16)
    h = a.numel()
    call("spark_add_rmsnorm", _p(a), _p(b), _p(gamma), float(eps), h, _p(res_out), _p(y), _stream())
    return y


def silu_mul_out(g, u, out):
    _cuda(g, "g", BF16)
    _cuda(u, "u", BF16)
    call("spark_silu_mul", _p(g), _p(u), g.numel(), _p(out), _stream())
    return out


def rope_neox_(x, cos_sin, pos):
    _cuda(x, "x", BF16)
    nh, dim = x.shape[-2], x.shape[-1]
    call("spark_rope_neox", _p(x), nh, dim, _p(cos_sin), _p(pos), _stream())
    return x


def add_rmsnorm_rows(a: torch.Tensor, b: torch.Tensor | None, gamma: torch.Tensor, eps: float):
    """Prefill rows: a / b bf16 [n, h] -> (bf16(a + b), bf16 RMSNorm(a + b) * gamma)."""
    _cuda(a, "a", BF16)
    _cuda(gamma, "gamma", BF16)
    n, h = a.shape
    a = a.contiguous()
    b = None if b is None else b.contiguous()
    res, y = torch.empty_like(a), torch.empty_like(a)
    call("spark_add_rmsnorm_rows", _p(a), _p(b), _p(gamma), float(eps), n, h, _p(res), _p(y), _stream())
    return res, y


def rope_rows_(x: torch.Tensor, nh: int, head_dim: int, rotary_dim: int, cos_sin: torch.Tensor, pos0: int):
    """In-place RoPE of the first ``nh`` heads of each row of x (bf16 [n, >= nh * head_dim],
    rows contiguous), row r at position pos0 + r."""
    _cuda(x, "x", BF16)
    _check(x.dim() == 2 and x.stride(1) == 1, "x must be [rows, cols] with contiguous rows")
    call("spark_rope_neox_rows", _p(x), x.stride(0), x.shape[0], nh, head_dim, rotary_dim, _p(cos_sin), pos0,
         _stream())
    return x


def act_mul_rows(gu: torch.Tensor, gelu_table: torch.Tensor | None = None) -> torch.Tensor:
    """gu bf16 [n, 2 I] (gate | up) -> bf16 [n, I] = act(gate) * up (SiLU, or GELU by the
    table of ``step.gelu_table``), the decode epilogues' arithmetic."""
    _cuda(gu, "gu", BF16)
    n, i2 = gu.shape
    gu = gu.contiguous()
    out = torch.empty((n, i2 // 2), dtype=BF16, device=gu.device)
    call("spark_act_mul_rows", _p(gu), n, i2 // 2, _p(gelu_table), _p(out), _stream())
    return out


def slot_mapping_out(num_tokens, query_start, positions, block_table, block_size, out):
    _cuda(out, "out", torch.int64)
    call("spark_slot_mapping", num_tokens, out.numel(), _p(query_start), _p(positions), _p(block_table), block_size,
         _p(out), _stream())
    return out


def kv_store_(k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor, k_cache: torch.Tensor,
              v_cache: torch.Tensor) -> None:
    """Scatter k / v [tokens, nkv, D] into the paged caches [blocks, nkv, bs, D] at
    slot_mapping (int64; negative slots skipped)."""
    _cuda(k, "k", BF16)
    _cuda(v, "v", BF16)
    _cuda(slot_mapping, "slot_mapping", torch.int64)
    _cuda(k_cache, "k_cache", BF16)
    _cuda(v_cache, "v_cache", BF16)
    t, nkv, d = k.shape
    _check(k_cache.dim() == 4 and k_cache.shape[1] == nkv and k_cache.shape[3] == d, "k_cache shape")
    call("spark_kv_store", _p(k.contiguous()), _p(v.contiguous()), _p(slot_mapping.contiguous()), t, nkv, d,
         k_cache.shape[2], _p(k_cache), _p(v_cache), _stream())


# ---------------------------------------------------------------- batches over the paged cache
# error-word bits of these operators (include/spark_b200.h)
ERR_WAIT, ERR_LENGTH, ERR_NO_PAGES, ERR_TABLE_WIDTH, ERR_NO_ROWS = 1, 4, 8, 16, 32
ERR_PAGE, ERR_POSITION, ERR_SLOT, ERR_PLAN = 64, 128, 256, 512


# the C interface's sizes are 32-bit; ctypes drops what is above them without a word
_INT_MAX = (1 << 31) - 1

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _launch(dev: int, name: str, *args) -> None:
    """Launch on device ``dev`` (the tensors' own), on its current stream.  Pointers are
    passed as integers and the checks below build no message before one fails: these
    calls are made per layer and step, where host time counts."""
    if dev == _current_device():
        call(name, *args, _raw_stream(dev))
        return
    with torch.cuda.device(dev):
        call(name, *args, _raw_stream(dev))


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, dev: int) -> None:
    """t must be a dense ``dtype`` tensor on CUDA device ``dev``."""
    if t.dtype is dtype and t.get_device() == dev and t.is_contiguous():
        return
    _cuda(t, name, dtype)
    raise ValueError(f"{name} must be on cuda:{dev}, got {t.device}")


def _need_all(dev: int, dtype: torch.dtype, tensors, names) -> None:
    """``_need`` of several tensors (in one loop: 0.1 us a tensor instead of 0.2)."""
    for t in tensors:
        if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
            for u, name in zip(tensors, names):
                _need(u, name, dtype, dev)


def _home(t: torch.Tensor, name: str, dtype: torch.dtype) -> int:
    """The CUDA device index of ``t``, which must have ``dtype``."""
    if not t.is_cuda or t.dtype is not dtype:
        raise ValueError(f"{name} must be a CUDA {dtype} tensor, got {t.dtype} on {t.device}")
    return t.get_device()


def _block_table(t: torch.Tensor, reqs: int, dev: int) -> None:
    if t.dtype is not torch.int32 or t.get_device() != dev:
        raise ValueError(f"block_table must be an int32 tensor on cuda:{dev}, got {t.dtype} on {t.device}")
    if t.dim() != 2 or t.stride(1) != 1 or t.shape[0] < reqs or t.shape[1] < 1:
        raise ValueError(f"block_table must be [{reqs} requests, pages] with dense rows, got {tuple(t.shape)}")


def paged_plan_out(ctx_lens, new_lens, block_table, block_size, query_start, seq_lens, positions, slot_mapping,
                   counter, error, free_blocks=None, free_head=None, free_head_out=None):
    """Block tables, token positions and slot maps of a batch from its request lengths, in
    one launch on the device.  ``ctx_lens`` / ``new_lens`` int32 [R]: cached and new tokens;
    writes ``query_start`` int32 [R + 1], ``seq_lens`` int32 [R], ``positions`` and
    ``slot_mapping`` int64 [rows] (rows behind the last token: 0 and -1) and, given
    ``free_blocks`` (int32 [F]) with ``free_head`` (int32 [1], ids taken so far), the new
    pages' ids into ``block_table`` and the advanced head into ``free_head_out`` (default:
    ``free_head`` itself).  All or nothing: a batch that does not fit comes out empty, with
    the reason in ``error`` (ERR_* bits).  ``counter`` int32 [1], zero before the first call
    and left zero; calls that may overlap on the device need one each.  No output may overlap
    an input or another output."""
    i32 = torch.int32
    dev = _home(ctx_lens, "ctx_lens", i32)
    R, rows = ctx_lens.numel(), positions.numel()
    _need_all(dev, i32, (ctx_lens, new_lens, query_start, seq_lens, counter, error),
              ("ctx_lens", "new_lens", "query_start", "seq_lens", "counter", "error"))
    _need_all(dev, torch.int64, (positions, slot_mapping), ("positions", "slot_mapping"))
    if R < 1 or new_lens.numel() != R or seq_lens.numel() != R or query_start.numel() != R + 1:
        raise ValueError("ctx_lens, new_lens and seq_lens hold one entry per request, query_start one more")
    if slot_mapping.numel() != rows:
        raise ValueError("positions and slot_mapping must have the same length")
    if counter.numel() < 1 or error.numel() < 1:
        raise ValueError("counter and error must hold one int32")
    num_free = 0 if free_blocks is None else free_blocks.numel()
    if rows > _INT_MAX or block_size > _INT_MAX or num_free > _INT_MAX:
        raise ValueError("rows, block_size and free_blocks must be below 2^31")
    _block_table(block_table, R, dev)
    if (free_blocks is None) != (free_head is None) or (free_head_out is not None and free_head is None):
        raise ValueError("give free_blocks and free_head together (and free_head_out only with them)")
    if free_blocks is not None:
        free_head_out = free_head if free_head_out is None else free_head_out
        _need_all(dev, i32, (free_blocks, free_head, free_head_out), ("free_blocks", "free_head", "free_head_out"))
        if free_head.numel() != 1 or free_head_out.numel() != 1:
            raise ValueError("free_head must hold one int32")
    width = block_table.shape[1]
    _launch(dev, "spark_paged_plan", ctx_lens.data_ptr(), new_lens.data_ptr(), R, _ptr(free_blocks),
            num_free, _ptr(free_head), _ptr(free_head_out),
            block_table.data_ptr(), block_table.stride(0) if R > 1 else width, width, int(block_size), rows,
            query_start.data_ptr(), seq_lens.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(),
            counter.data_ptr(), error.data_ptr())


def qk_norm_rope_store_rows(qkv, nq, nkv, head_dim, q_gamma, k_gamma, eps, cos_sin, positions, slot_mapping, k_cache,
                            v_cache, q_out, error):
    """Rows of a fused qkv output (bf16 [rows, >= (nq + 2 nkv) * head_dim], rows dense) in one
    pass: per-head RMS norm of q and k (``q_gamma`` / ``k_gamma`` bf16 [head_dim], or both
    None), rotation at ``positions`` (int64 [rows]) by ``cos_sin`` bf16 [max_pos,
    rotary_dim], q to ``q_out`` bf16 [rows, nq, head_dim] and k, v to the paged caches at
    ``slot_mapping`` (int64 [rows], negative: not stored; no slot twice).  fp32 inside, one
    rounding."""
    dev = _home(qkv, "qkv", BF16)
    if qkv.dim() != 2 or (qkv.stride(1) != 1 and qkv.shape[1] != 1) or qkv.shape[1] < (nq + 2 * nkv) * head_dim:
        raise ValueError(f"qkv must be [rows, >= {(nq + 2 * nkv) * head_dim}] with dense rows, got {tuple(qkv.shape)}")
    rows = qkv.shape[0]
    _need_all(dev, BF16, (cos_sin, k_cache, v_cache, q_out), ("cos_sin", "k_cache", "v_cache", "q_out"))
    _need_all(dev, torch.int64, (positions, slot_mapping), ("positions", "slot_mapping"))
    _need(error, "error", torch.int32, dev)
    if positions.numel() < rows or slot_mapping.numel() < rows:
        raise ValueError("positions and slot_mapping must hold one entry per row")
    if error.numel() < 1:
        raise ValueError("error must hold one int32")
    if (q_gamma is None) != (k_gamma is None):
        raise ValueError("give q_gamma and k_gamma together")
    if q_gamma is not None:
        _need_all(dev, BF16, (q_gamma, k_gamma), ("q_gamma", "k_gamma"))
        if q_gamma.numel() != head_dim or k_gamma.numel() != head_dim:
            raise ValueError("q_gamma and k_gamma must hold head_dim values")
    if cos_sin.dim() != 2:
        raise ValueError("cos_sin must be [max_pos, rotary_dim]")
    ks = k_cache.shape
    if len(ks) != 4 or v_cache.shape != ks or ks[1] != nkv or ks[3] != head_dim:
        raise ValueError("caches must be [blocks, nkv, block_size, head_dim]")
    if q_out.numel() != rows * nq * head_dim:
        raise ValueError("q_out must be [rows, nq, head_dim]")
    _launch(dev, "spark_qk_norm_rope_store_rows", qkv.data_ptr(), qkv.stride(0) if rows > 1 else
            (qkv.shape[1] + 7) // 8 * 8, rows, nq, nkv, head_dim, _ptr(q_gamma), _ptr(k_gamma), eps,
            cos_sin.data_ptr(), cos_sin.shape[0], cos_sin.shape[1], positions.data_ptr(), slot_mapping.data_ptr(),
            ks[2], ks[0], k_cache.data_ptr(), v_cache.data_ptr(), q_out.data_ptr(), error.data_ptr())
    return q_out


class AttnPlan:
    """Work list and workspace of the paged attention for one head layout and window.

    ``update`` (packed prompts, chunks, single tokens) or ``update_prefix`` (one token per
    request behind a common prefix) makes the list from device tensors, without a host
    copy, once per step; every layer of that layout then uses it.  Both can be captured
    into a CUDA graph, which holds the plan's addresses: the plan has to live as long as the
    graph.  Calls that may overlap on the device need a plan each: the plan and the partial
    results are overwritten by the next one.  ``error`` int32 [1] collects what
    ``update`` found (ERR_* bits)."""

    def __init__(self, max_tokens: int, max_reqs: int, nq: int, nkv: int, head_dim: int, device="cuda",
                 window: int = 0):
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        _check(device.type == "cuda", "the plan lives on a CUDA device")
        _check(0 <= window <= _INT_MAX, "window must be positive and below 2^31, or 0 for none")
        _check(max(max_tokens, max_reqs, nq, nkv, head_dim) <= _INT_MAX, "sizes must be below 2^31")
        nbytes = lib().spark_attn_plan_bytes(max_tokens, max_reqs, nq, nkv, head_dim)
        _check(nbytes > 0, f"unsupported attention shape: {max_tokens} tokens, {max_reqs} requests, {nq} query / "
                           f"{nkv} kv heads of {head_dim}")
        rows = lib().spark_attn_part_rows(max_tokens, max_reqs, nq, nkv, head_dim)
        self.max_tokens, self.max_reqs, self.window = int(max_tokens), int(max_reqs), int(window)
        self.nq, self.nkv, self.head_dim, self.device = nq, nkv, head_dim, device
        self.dev = device.index
        self.buf = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        self.part_o = torch.empty((rows, nkv, head_dim), dtype=torch.float32, device=device)
        self.part_ml = torch.empty((rows, nkv, 2), dtype=torch.float32, device=device)
        self.error = torch.zeros(1, dtype=torch.int32, device=device)
        self.kind, self.reqs = None, 0

    def _make(self, kind, reqs, query_start, seq_lens, prefix_len):
        if reqs > self.max_reqs:
            raise ValueError(f"{reqs} requests in a plan for {self.max_reqs}")
        _launch(self.dev, "spark_attn_plan", _ptr(query_start), _ptr(seq_lens), _ptr(prefix_len), reqs,
                self.max_tokens, self.max_reqs, self.nq, self.nkv, self.head_dim, self.window, _ptr(self.buf),
                _ptr(self.error))
        self.kind, self.reqs = kind, reqs
        return self

    def update(self, query_start: torch.Tensor, seq_lens: torch.Tensor) -> "AttnPlan":
        """A packed batch: request r's query tokens are rows query_start[r] ..
        query_start[r + 1] - 1 (int32 [R + 1]), the last of its seq_lens[r] (int32 [R]) keys."""
        _need(query_start, "query_start", torch.int32, self.dev)
        _need(seq_lens, "seq_lens", torch.int32, self.dev)
        reqs = seq_lens.numel()
        _check(reqs >= 1 and query_start.numel() == reqs + 1, "query_start must have one entry more than seq_lens")
        return self._make("prompt", reqs, query_start, seq_lens, None)

    def update_prefix(self, seq_lens: torch.Tensor, prefix_len: torch.Tensor) -> "AttnPlan":
        """One query token per request, seq_lens[r] (int32 [R]) keys each, the first
        prefix_len (int32 [1]) of them the same for all."""
        _need(seq_lens, "seq_lens", torch.int32, self.dev)
        _need(prefix_len, "prefix_len", torch.int32, self.dev)
        _check(self.window == 0, "a shared prefix is read without a window")
        _check(prefix_len.numel() == 1, "prefix_len must hold one int32")
        reqs = seq_lens.numel()
        _check(1 <= reqs <= self.max_tokens, f"{reqs} requests in a plan for {self.max_tokens} tokens")
        return self._make("prefix", reqs, None, seq_lens, prefix_len)


def _heads(t: torch.Tensor, name: str, plan: AttnPlan) -> None:
    shape = t.shape
    if t.dtype is not BF16 or t.get_device() != plan.dev:
        raise ValueError(f"{name} must be a bfloat16 tensor on cuda:{plan.dev}, got {t.dtype} on {t.device}")
    if len(shape) != 3 or shape[1] != plan.nq or shape[2] != plan.head_dim or (t.stride(2) != 1 and t.numel()):
        raise ValueError(f"{name} must be [tokens, {plan.nq}, {plan.head_dim}], heads dense, got {tuple(shape)}")


def _attn_paged(kind, q, k_cache, v_cache, block_table, plan, scale, out, error, wait_ns):
    if plan.kind != kind:
        raise ValueError(f"the plan was made for {plan.kind!r}, not {kind!r}")
    nq, nkv, D, dev = plan.nq, plan.nkv, plan.head_dim, plan.dev
    _heads(q, "q", plan)
    _heads(out, "out", plan)
    tokens = q.shape[0]
    if out.shape[0] < tokens or tokens > plan.max_tokens:
        raise ValueError(f"{tokens} tokens: out has {out.shape[0]} rows, the plan room for {plan.max_tokens}")
    _need_all(dev, BF16, (k_cache, v_cache), ("k_cache", "v_cache"))
    ks = k_cache.shape
    if len(ks) != 4 or v_cache.shape != ks or ks[1] != nkv or ks[3] != D:
        raise ValueError(f"caches must be [blocks, {nkv}, block_size, {D}]")
    _block_table(block_table, plan.reqs, dev)
    _need(error, "error", torch.int32, dev)
    if error.numel() < 1:
        raise ValueError("error must hold one int32")
    qt, qh, _ = q.stride()
    ot, oh, _ = out.stride()
    _launch(dev, "spark_attn_paged_bounded", q.data_ptr(), qt, qh, tokens, k_cache.data_ptr(), v_cache.data_ptr(),
            ks[0], ks[2], block_table.data_ptr(), block_table.stride(0), block_table.shape[1], block_table.shape[0],
            plan.max_tokens, plan.max_reqs, nq, nkv, D, plan.window, scale, plan.buf.data_ptr(), plan.part_o.data_ptr(),
            plan.part_ml.data_ptr(), out.data_ptr(), ot, oh, error.data_ptr(), wait_ns)
    return out


def attn_prompt_out(q, k_cache, v_cache, block_table, plan: AttnPlan, scale, out, error, wait_ns: int = -1):
    """Causal attention of a packed batch over the paged caches (``plan.update`` made this
    step's list): q / out bf16 [tokens, nq, D] (any token and head strides that are
    multiples of 8), caches bf16 [blocks, nkv, block_size, D], block_table int32 [R, pages].
    Whole prompts, chunks on top of cached context and single tokens alike; tokens without
    keys give zero, rows of ``out`` behind the last planned token are left as they were.
    Scores and sums are fp32, the probabilities are rounded to bf16 as an operand of the product
    with V.  Values at positions a request does hold must be finite; what its pages carry past
    its length does not matter.  A row that sees a NaN or +inf score is NaN.  ``error`` (int32
    [1], required): nonzero, out is not valid (ERR_* bits)."""
    return _attn_paged("prompt", q, k_cache, v_cache, block_table, plan, scale, out, error, wait_ns)


def attn_shared_prefix_out(q, k_cache, v_cache, block_table, plan: AttnPlan, scale, out, error, wait_ns: int = -1):
    """Attention of one query token per request (q / out bf16 [R, nq, D]) where all requests
    share their first positions (``plan.update_prefix``): the prefix's pages are read once
    for the whole batch, through the first request's table (which must hold as much of it as
    the longest request has), each request's own keys through its own; the parts join by
    log-sum-exp.  Otherwise as ``attn_prompt_out``."""
    _check(q.shape[0] >= plan.reqs, "q must have a row per request")
    return _attn_paged("prefix", q, k_cache, v_cache, block_table, plan, scale, out, error, wait_ns)


def set_pdl(enabled: bool) -> None:
    call("spark_set_pdl", 1 if enabled else 0)


def set_gemv_ring(enabled: bool) -> None:
    """Choose the weight-ring GEMV (default) or the register-direct GEMV for K % 512 == 0."""
    call("spark_set_gemv_ring", 1 if enabled else 0)


def read_device_error(reset: bool = True) -> int:
    """Synchronously read (and optionally clear) the library's device error word."""
    v = ctypes.c_int(0)
    call("spark_read_device_error", ctypes.byref(v), 1 if reset else 0)
    return int(v.value)


# ---------------------------------------------------------------- torch.library custom ops
@torch.library.custom_op("spark_b200::q4_gemv", mutates_args=())
def _op_q4_gemv(x: torch.Tensor, qs: torch.Tensor, d: torch.Tensor) -> torch.Tensor:
    return q4_gemv(x.contiguous(), qs, d)


@_op_q4_gemv.register_fake
def _(x, qs, d):
    return x.new_empty((*x.shape[:-1], qs.shape[0]))


@torch.library.custom_op("spark_b200::rmsnorm_q4_gemv", mutates_args=())
def _op_rmsnorm_q4_gemv(a: torch.Tensor, b: torch.Tensor | None, gamma: torch.Tensor, eps: float,
                        qs: torch.Tensor, d: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    y = a.new_empty((qs.shape[0],))
    res = torch.empty_like(a)
    rmsnorm_q4_gemv_out(a.contiguous(), None if b is None else b.contiguous(), gamma, eps, qs, d, y, res)
    return y, res


@_op_rmsnorm_q4_gemv.register_fake
def _(a, b, gamma, eps, qs, d):
    return a.new_empty((qs.shape[0],)), torch.empty_like(a)


@torch.library.custom_op("spark_b200::rmsnorm_gate_up_silu", mutates_args=())
def _op_gate_up(a: torch.Tensor, b: torch.Tensor | None, gamma: torch.Tensor, eps: float, qs: torch.Tensor,
                d: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    mid = a.new_empty((qs.shape[0] // 2,))
    res = torch.empty_like(a)
    rmsnorm_gate_up_silu_out(a.contiguous(), None if b is None else b.contiguous(), gamma, eps, qs, d, mid, res)
    return mid, res


@_op_gate_up.register_fake
def _(a, b, gamma, eps, qs, d):
    return a.new_empty((qs.shape[0] // 2,)), torch.empty_like(a)


@torch.library.custom_op("spark_b200::qkv_rope_kvstore", mutates_args=("k_cache", "v_cache"))
def _op_qkv(a: torch.Tensor, b: torch.Tensor | None, gamma: torch.Tensor, eps: float, qs: torch.Tensor,
            d: torch.Tensor, nq: int, nkv: int, head_dim: int, cos_sin: torch.Tensor, pos: torch.Tensor,
            slot_mapping: torch.Tensor, block_size: int, k_cache: torch.Tensor,
            v_cache: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    q = a.new_empty((nq, head_dim))
    res = torch.empty_like(a)
    qkv_rope_kvstore_out(a.contiguous(), None if b is None else b.contiguous(), gamma, eps, qs, d, nq, nkv,
                         head_dim, cos_sin, pos, None, slot_mapping, block_size, k_cache, v_cache, q, res)
    return q, res


@_op_qkv.register_fake
def _(a, b, gamma, eps, qs, d, nq, nkv, head_dim, cos_sin, pos, slot_mapping, block_size, k_cache, v_cache):
    return a.new_empty((nq, head_dim)), torch.empty_like(a)


@torch.library.custom_op("spark_b200::attn_decode", mutates_args=())
def _op_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
             seq_len: torch.Tensor, splits: int, max_split_tokens: int, scale: float) -> torch.Tensor:
    nq, dim = q.shape[-2], q.shape[-1]
    part_o = torch.empty((splits, nq, dim), dtype=torch.float32, device=q.device)
    part_lse = torch.empty((splits, nq), dtype=torch.float32, device=q.device)
    attn_splitkv_out(q.contiguous(), k_cache, v_cache, block_table, splits, max_split_tokens, scale, part_o, part_lse,
                     seq_len=seq_len)
    out = q.new_empty((nq, dim))
    attn_combine_out(part_o, part_lse, out)
    return out


@_op_attn.register_fake
def _(q, k_cache, v_cache, block_table, seq_len, splits, max_split_tokens, scale):
    return q.new_empty((q.shape[-2], q.shape[-1]))


@torch.library.custom_op("spark_b200::add_rmsnorm", mutates_args=())
def _op_add_rmsnorm(a: torch.Tensor, b: torch.Tensor | None, gamma: torch.Tensor,
                    eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    y = torch.empty_like(a)
    res = torch.empty_like(a)
    add_rmsnorm_out(a.contiguous(), None if b is None else b.contiguous(), gamma, eps, y, res)
    return y, res


@_op_add_rmsnorm.register_fake
def _(a, b, gamma, eps):
    return torch.empty_like(a), torch.empty_like(a)


@torch.library.custom_op("spark_b200::silu_mul", mutates_args=())
def _op_silu_mul(gu: torch.Tensor) -> torch.Tensor:
    half = gu.shape[-1] // 2
    g = gu[..., :half].contiguous()
    u = gu[..., half:].contiguous()
    out = torch.empty_like(g)
    silu_mul_out(g, u, out)
    return out


@_op_silu_mul.register_fake
def _(gu):
    return gu.new_empty((*gu.shape[:-1], gu.shape[-1] // 2))


@torch.library.custom_op("spark_b200::qk_norm_rope_store_rows", mutates_args=("k_cache", "v_cache", "error"))
def _op_qk_rows(qkv: torch.Tensor, nq: int, nkv: int, head_dim: int, q_gamma: torch.Tensor | None,
                k_gamma: torch.Tensor | None, eps: float, cos_sin: torch.Tensor, positions: torch.Tensor,
                slot_mapping: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                error: torch.Tensor) -> torch.Tensor:
    q = qkv.new_empty((qkv.shape[0], nq, head_dim))
    return qk_norm_rope_store_rows(qkv, nq, nkv, head_dim, q_gamma, k_gamma, eps, cos_sin, positions, slot_mapping,
                                   k_cache, v_cache, q, error)


@_op_qk_rows.register_fake
def _(qkv, nq, nkv, head_dim, q_gamma, k_gamma, eps, cos_sin, positions, slot_mapping, k_cache, v_cache, error):
    return qkv.new_empty((qkv.shape[0], nq, head_dim))


@torch.library.custom_op("spark_b200::attn_prompt", mutates_args=("error",))
def _op_attn_prompt(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    query_start: torch.Tensor, seq_lens: torch.Tensor, scale: float, window: int,
                    error: torch.Tensor) -> torch.Tensor:
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    if q.shape[0] == 0:
        return out
    plan = AttnPlan(q.shape[0], seq_lens.numel(), q.shape[1], k_cache.shape[1], q.shape[2], q.device, window)
    plan.update(query_start, seq_lens)
    attn_prompt_out(q, k_cache, v_cache, block_table, plan, scale, out, error)
    error.bitwise_or_(plan.error)
    return out


@_op_attn_prompt.register_fake
def _(q, k_cache, v_cache, block_table, query_start, seq_lens, scale, window, error):
    return q.new_empty(q.shape)


@torch.library.custom_op("spark_b200::attn_shared_prefix", mutates_args=("error",))
def _op_attn_prefix(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, prefix_len: torch.Tensor, scale: float,
                    error: torch.Tensor) -> torch.Tensor:
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    if q.shape[0] == 0:
        return out
    plan = AttnPlan(q.shape[0], seq_lens.numel(), q.shape[1], k_cache.shape[1], q.shape[2], q.device)
    plan.update_prefix(seq_lens, prefix_len)
    attn_shared_prefix_out(q, k_cache, v_cache, block_table, plan, scale, out, error)
    error.bitwise_or_(plan.error)
    return out


@_op_attn_prefix.register_fake
def _(q, k_cache, v_cache, block_table, seq_lens, prefix_len, scale, error):
    return q.new_empty(q.shape)


def q6k_dequantize(blocks: torch.Tensor) -> torch.Tensor:
    """gguf Q6_K super-blocks (uint8 [..., 210] on the device) -> fp32 weights, the decode
    of gguf 0.19.0 (``spark_q6k_dequantize``)."""
    b = blocks.contiguous()
    if b.dtype != torch.uint8 or b.numel() % 210:
        raise ValueError("Q6_K blocks are uint8 rows of 210-byte super-blocks")
    nb = b.numel() // 210
    out = torch.empty(nb * 256, dtype=torch.float32, device=b.device)
    call("spark_q6k_dequantize", _p(b), nb, _p(out), _stream())
    return out
