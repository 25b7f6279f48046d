"""CPU checks of the paged-batch entry points: sizes, strides, alignments and missing
pointers are refused on the host, before any launch (no device work is issued)."""
from __future__ import annotations

import ctypes

import pytest

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first
OFF = ctypes.c_void_p(0x1008)
INVALID, SHAPE, ALIGN, LARGE = 1, 2, 3, 5


@pytest.fixture(scope="module")
def L():
    import spark_b200
    from spark_b200 import _lib

    spark_b200.ensure_built()
    return _lib.lib()


def _plan(L, **k):
    a = dict(ctx=FAKE, new=FAKE, reqs=4, free=FAKE, num_free=9, head=FAKE, head_out=FAKE, table=FAKE, stride=8,
             width=8, bs=16, rows=0, qs=FAKE, sl=FAKE, pos=None, slots=None, counter=FAKE, error=FAKE, stream=None)
    a.update(k)
    return L.spark_paged_plan(*a.values())


@pytest.mark.parametrize("bad,status", [
    (dict(ctx=None), INVALID), (dict(error=None), INVALID), (dict(counter=None), INVALID), (dict(rows=5), INVALID),
    (dict(head=None), INVALID), (dict(free=None), INVALID), (dict(head_out=None), INVALID), (dict(reqs=0), SHAPE),
    (dict(reqs=-3), SHAPE), (dict(rows=-1), SHAPE), (dict(bs=0), SHAPE), (dict(width=0), SHAPE),
    (dict(stride=7), SHAPE), (dict(num_free=-1), SHAPE), (dict(reqs=8193), LARGE),
    (dict(qs=OFF), INVALID), (dict(sl=OFF), INVALID)])  # (seq_lens / query_start in the place of the lengths)
def test_paged_plan_refuses(L, bad, status):
    assert _plan(L, **bad) == status


def _rows(L, **k):
    a = dict(qkv=FAKE, stride=1536, rows=4, nq=8, nkv=2, D=128, qg=FAKE, kg=FAKE, eps=ctypes.c_float(1e-6), cs=FAKE,
             max_pos=100, rot=128, pos=FAKE, slots=FAKE, bs=16, blocks=4, kc=FAKE, vc=FAKE, q=FAKE, error=FAKE,
             stream=None)
    a.update(k)
    return L.spark_qk_norm_rope_store_rows(*a.values())


@pytest.mark.parametrize("bad,status", [
    (dict(qkv=None), INVALID), (dict(q=None), INVALID), (dict(error=None), INVALID), (dict(qg=None), INVALID),
    (dict(kg=None), INVALID), (dict(cs=None), INVALID), (dict(D=64), SHAPE), (dict(rot=0), SHAPE),
    (dict(rot=24), SHAPE), (dict(rot=144), SHAPE), (dict(stride=1528), SHAPE), (dict(rows=-1), SHAPE),
    (dict(nkv=0), SHAPE), (dict(blocks=0), SHAPE), (dict(max_pos=0), SHAPE), (dict(stride=1540), ALIGN),
    (dict(qkv=OFF), ALIGN), (dict(kc=OFF), ALIGN), (dict(q=OFF), ALIGN), (dict(kg=OFF), ALIGN)])
def test_rope_store_refuses(L, bad, status):
    assert _rows(L, **bad) == status


def test_attn_plan_sizes_too_large_are_refused(L):
    for fn in (L.spark_attn_plan_bytes, L.spark_attn_part_rows):
        assert fn(1 << 16, 1 << 16, 128, 128, 128) == -1  # rows to join past 2^30
        assert fn(1 << 16, 1 << 15, 32, 8, 128) > 0
        assert fn((1 << 22) + 1, 1, 32, 8, 128) == -1


def test_rope_store_of_no_rows_is_no_work(L):
    assert _rows(L, rows=0, qkv=None, q=None) == 0


def test_attn_plan_sizes(L):
    assert L.spark_attn_plan_bytes(1, 1, 32, 8, 128) > 0 and L.spark_attn_plan_bytes(1, 1, 32, 8, 128) % 16 == 0
    assert L.spark_attn_part_rows(4096, 16, 32, 8, 128) > 0
    for shape in ((0, 1, 8, 2, 128), (1, 0, 8, 2, 128), (1, 1, 8, 3, 128), (1, 1, 8, 2, 96), (1, 1, 258, 2, 128),
                  ((1 << 22) + 1, 1, 8, 2, 128), (1, (1 << 16) + 1, 8, 2, 128)):
        assert L.spark_attn_plan_bytes(*shape) == -1 and L.spark_attn_part_rows(*shape) == -1


def _make(L, **k):
    a = dict(qs=FAKE, sl=FAKE, prefix=None, reqs=2, tokens=64, max_reqs=4, nq=8, nkv=2, D=128, window=0, plan=FAKE,
             error=FAKE, stream=None)
    a.update(k)
    return L.spark_attn_plan(*a.values())


@pytest.mark.parametrize("bad,status", [
    (dict(qs=None), INVALID), (dict(prefix=FAKE), INVALID), (dict(sl=None), INVALID), (dict(plan=None), INVALID),
    (dict(error=None), INVALID), (dict(reqs=5), SHAPE), (dict(reqs=-1), SHAPE), (dict(window=-1), SHAPE),
    (dict(qs=None, prefix=FAKE, window=3), SHAPE), (dict(qs=None, prefix=FAKE, reqs=4, tokens=3), SHAPE),
    (dict(D=64), SHAPE), (dict(plan=OFF), ALIGN)])
def test_attn_plan_refuses(L, bad, status):
    assert _make(L, **bad) == status


def _attn(L, **k):
    a = dict(q=FAKE, qt=1024, qh=128, tokens=10, kc=FAKE, vc=FAKE, blocks=4, bs=16, table=FAKE, ts=8, tw=8,
             max_tokens=64, max_reqs=4, nq=8, nkv=2, D=128, window=0, scale=ctypes.c_float(0.1), plan=FAKE, po=FAKE,
             ml=FAKE, out=FAKE, ot=1024, oh=128, error=FAKE, wait=-1, stream=None)
    a.update(k)
    return L.spark_attn_paged(*a.values())


@pytest.mark.parametrize("bad,status", [
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(kc=None), INVALID), (dict(plan=None), INVALID),
    (dict(error=None), INVALID), (dict(po=None), INVALID), (dict(tokens=65), SHAPE), (dict(tokens=-1), SHAPE),
    (dict(bs=8), SHAPE), (dict(bs=24), SHAPE), (dict(blocks=0), SHAPE), (dict(tw=0), SHAPE), (dict(window=-2), SHAPE),
    (dict(scale=ctypes.c_float(0.0)), SHAPE), (dict(scale=ctypes.c_float(-1.0)), SHAPE),
    (dict(scale=ctypes.c_float(float("nan"))), SHAPE), (dict(scale=ctypes.c_float(float("inf"))), SHAPE),
    (dict(nq=7), SHAPE), (dict(D=192), SHAPE), (dict(blocks=1 << 28), LARGE), (dict(qt=1020), ALIGN),
    (dict(oh=132), ALIGN), (dict(q=OFF), ALIGN), (dict(out=OFF), ALIGN), (dict(vc=OFF), ALIGN)])
def test_attn_paged_refuses(L, bad, status):
    assert _attn(L, **bad) == status


def test_attn_paged_of_no_tokens_is_no_work(L):
    assert _attn(L, tokens=0, q=None, out=None) == 0


def test_wrappers_refuse_host_tensors():
    import torch
    from spark_b200 import ops

    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_plan_out(i, i, i.view(1, 2), 16, i, i, i.long(), i.long(), i, i)
    x = torch.zeros((2, 384), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_store_rows(x, 1, 1, 128, None, None, 1e-6, x, i.long(), i.long(), x, x, x, i)
    with pytest.raises(ValueError):
        ops.AttnPlan(4, 1, 8, 2, 128, device="cpu")


def test_paged_custom_ops_trace_on_meta_tensors():
    import torch
    from spark_b200 import ops  # noqa: F401

    bf = {"dtype": torch.bfloat16, "device": "meta"}
    i32 = {"dtype": torch.int32, "device": "meta"}
    q, c = torch.empty((5, 8, 128), **bf), torch.empty((4, 2, 16, 128), **bf)
    t, s, e = torch.empty((2, 3), **i32), torch.empty(2, **i32), torch.empty(1, **i32)
    assert torch.ops.spark_b200.attn_prompt(q, c, c, t, torch.empty(3, **i32), s, 0.1, 0, e).shape == (5, 8, 128)
    assert torch.ops.spark_b200.attn_shared_prefix(q, c, c, t, s, e, 0.1, e).shape == (5, 8, 128)
    p = torch.empty(5, dtype=torch.int64, device="meta")
    y = torch.ops.spark_b200.qk_norm_rope_store_rows(torch.empty((5, 1536), **bf), 8, 2, 128, None, None, 1e-6,
                                                     torch.empty((9, 128), **bf), p, p, c, c.clone(), e)
    assert y.shape == (5, 8, 128)


def test_rows_of_a_packed_prefill_are_dealt_in_order():
    from spark_b200.prefill import _next_rows
    assert _next_rows([130, 1, 77], 40) == [40, 0, 0]
    assert _next_rows([10, 1, 77], 40) == [10, 1, 29]
    assert _next_rows([0, 0, 5], 40) == [0, 0, 5]


def test_cascade_is_asked_for_only_where_it_serves(monkeypatch):
    pytest.importorskip("vllm")
    from spark_b200.plugin.attention import PAGED_ENV, SparkAttentionMetadataBuilder as B
    b = B.__new__(B)
    ask = lambda prefix=512, q=(1, 1, 1), **k: b.use_cascade_attention(  # noqa: E731
        prefix, list(q), 32, 8, k.get("alibi", False), k.get("sliding", False), k.get("local", False), 148,
        k.get("dcp", 1))
    monkeypatch.delenv(PAGED_ENV, raising=False)
    assert not ask()  # off unless switched on
    monkeypatch.setenv(PAGED_ENV, "1")
    assert ask()
    assert not ask(prefix=127) and not ask(q=(1,)) and not ask(q=(1, 2)) and not ask(alibi=True)
    assert not ask(sliding=True) and not ask(local=True) and not ask(dcp=2)
