"""Packed prefill (``spark_b200.prefill.prefill_packed``: paged_plan -> rows -> paged
attention) and the vLLM backend's paged path, against the paths they stand beside.

The packed path computes the layers of ``prefill`` with the same GEMMs, norms and
activations; its rotation is bit for bit the row kernel's, so layer 0's pages are equal to
``prefill``'s exactly, and what differs afterwards is the attention's bf16 rounding, carried
through the layers: the tolerance of the batched prefill against decode (3 %)."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


def _cfgs():
    from spark_b200.config import spark_x26_config, tiny_config
    return [tiny_config(num_layers=3),
            spark_x26_config(num_layers=4, hidden_size=512, num_q_heads=8, num_kv_heads=2, intermediate_size=1024,
                             vocab_size=4096, sliding_window=33, max_position=4096, name="spark-tiny")]


def _near(a, b):
    a, b = a.float(), b.float()
    assert (a - b).abs().max().item() <= 0.03 * a.abs().max().item() + 0.03


@pytest.mark.parametrize("gemm", ["q4", "bf16"])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("P,chunk", [(90, 64), (150, 8192), (1, 4)])
def test_paged_prefill_matches_sdpa_prefill(cuda, which, gemm, P, chunk):
    import torch
    from spark_b200.model import DecodeEngine, SyntheticWeights
    cfg = _cfgs()[which]
    w = SyntheticWeights(cfg, device="cuda", seed=11)
    prompt = (torch.arange(P, dtype=torch.int32) * 131 + 7) % cfg.vocab_size
    ref = DecodeEngine(w, max_seq_len=256, num_blocks=8, seed=11)
    ref.prefill_batched(prompt, chunk=chunk, gemm=gemm)
    eng = DecodeEngine(w, max_seq_len=256, num_blocks=8, seed=11)
    tok = eng.prefill_batched(prompt, chunk=chunk, gemm=gemm, attn="paged")
    torch.cuda.synchronize()
    pos = torch.arange(P, device="cuda")
    blk, off = eng.block_table[pos // cfg.block_size].long(), pos % cfg.block_size
    assert torch.equal(ref.k_cache[0][blk, :, off], eng.k_cache[0][blk, :, off])
    assert torch.equal(ref.v_cache[0][blk, :, off], eng.v_cache[0][blk, :, off])
    for li in range(cfg.num_layers):
        _near(ref.k_cache[li][blk, :, off], eng.k_cache[li][blk, :, off])
        _near(ref.v_cache[li][blk, :, off], eng.v_cache[li][blk, :, off])
    _near(ref.logits, eng.logits)
    assert int(eng.pos.item()) == P and int(tok) == int(torch.argmax(eng.logits.float()))
    for _ in range(3):  # decode goes on from the pages
        eng.step()
    torch.cuda.synchronize()
    assert int(eng.error.item()) == 0 and int(eng.pos.item()) == P + 3


def test_packed_prefill_of_a_batch_matches_one_by_one(cuda):
    """Four prompts of different lengths through BatchDecodeEngine, cut into uneven batches."""
    import torch
    from spark_b200.batch import BatchDecodeEngine
    from spark_b200.config import tiny_config
    from spark_b200.model import SyntheticWeights
    cfg = tiny_config(num_layers=2)
    w = SyntheticWeights(cfg, device="cuda", seed=5)
    lens = [130, 1, 77, 200]
    prompts = [[(37 * i + 11 * b) % cfg.vocab_size for i in range(n)] for b, n in enumerate(lens)]
    ref = BatchDecodeEngine(w, 4, max_seq_len=256, seed=5)
    ref.prefill(prompts)
    for chunk in (2048, 40):
        eng = BatchDecodeEngine(w, 4, max_seq_len=256, seed=5)
        tok = eng.prefill(prompts, chunk=chunk, packed=True)
        torch.cuda.synchronize()
        _near(ref.logits, eng.logits)
        assert eng.pos.tolist() == lens and tok.tolist() == torch.argmax(eng.logits.float(), -1).tolist()
        for b, n in enumerate(lens):
            pos = torch.arange(n, device="cuda")
            blk, off = eng.block_tables[b, pos // cfg.block_size].long(), pos % cfg.block_size
            assert torch.equal(ref.k_cache[0][blk, :, off], eng.k_cache[0][blk, :, off])
            _near(ref.v_cache[1][blk, :, off], eng.v_cache[1][blk, :, off])
        for _ in range(3):
            eng.step()
        torch.cuda.synchronize()
        assert int(eng.error.item()) == 0 and eng.pos.tolist() == [n + 3 for n in lens]


def test_packed_prefill_refuses(cuda):
    import torch
    from spark_b200.config import tiny_config
    from spark_b200.model import DecodeEngine, SyntheticWeights
    from spark_b200.prefill import prefill_packed
    w = SyntheticWeights(tiny_config(num_layers=1), device="cuda", seed=1)
    eng = DecodeEngine(w, max_seq_len=128, num_blocks=4)
    table = eng.block_table.view(1, -1)
    with pytest.raises(ValueError):
        eng.prefill_batched([1, 2], attn="flash")
    for bad in ([], [[]], [[1] * 129], [[1], [2]]):
        with pytest.raises(ValueError):
            prefill_packed(eng, bad, table)
    with pytest.raises(RuntimeError):  # a table that names a page outside the cache
        prefill_packed(eng, [[1, 2, 3]], torch.full_like(table, 1 << 20))


def _metadata(seq_lens, query_lens, table, slots, prefix=0):
    import torch
    from spark_b200.plugin.attention import SparkAttentionMetadata
    i32 = {"dtype": torch.int32}
    start = [0]
    for n in query_lens:
        start.append(start[-1] + n)
    return SparkAttentionMetadata(
        num_actual_tokens=start[-1], num_reqs=len(seq_lens), max_query_len=max(query_lens), max_seq_len=max(seq_lens),
        query_start_loc=torch.tensor(start, **i32).cuda(), query_start_loc_cpu=torch.tensor(start, **i32),
        seq_lens=torch.tensor(seq_lens, **i32).cuda(), block_table=table, slot_mapping=slots, splits=24,
        max_split_tokens=128, prefix_len=torch.tensor([prefix], **i32).cuda() if prefix else None)


@pytest.mark.parametrize("nq,nkv,D,window", [(32, 8, 128, None), (16, 4, 256, None), (16, 4, 256, 64)])
def test_backend_paged_prefill_matches_torch_path(cuda, monkeypatch, nq, nkv, D, window):
    """A mixed batch (a prompt, a chunk, a single token) through the backend with the paged
    path on, against the same call with it off; |diff| <= u sum p |v| + u |o| with |v| < 6."""
    vllm = pytest.importorskip("vllm")  # noqa: F841
    import torch
    from spark_b200.plugin.attention import PAGED_ENV, SparkAttentionImpl
    g = torch.Generator(device="cuda").manual_seed(3)
    bs, seq_lens, query_lens = 128, [200, 700, 333], [200, 60, 1]
    need = [-(-n // bs) for n in seq_lens]
    kv0 = torch.randn((2, sum(need) + 2, nkv, bs, D), generator=g, device="cuda").to(torch.bfloat16)
    perm = torch.randperm(sum(need) + 2, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((3, max(need)), dtype=torch.int32, device="cuda")
    at, slots = 0, []
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
        p = torch.arange(seq_lens[r] - query_lens[r], seq_lens[r], device="cuda")
        slots.append(table[r, p // bs].long() * bs + p % bs)
    slots = torch.cat(slots)
    T = sum(query_lens)
    q, k, v = (torch.randn((T, h * D), generator=g, device="cuda").to(torch.bfloat16) for h in (nq, nkv, nkv))
    outs = []
    for on in ("0", "1"):
        monkeypatch.setenv(PAGED_ENV, on)
        impl = SparkAttentionImpl(nq, D, 1 / math.sqrt(D), nkv, sliding_window=window)
        kv = kv0.clone()
        md = _metadata(seq_lens, query_lens, table, slots)
        out = torch.full((T + 5, nq * D), 9.0, dtype=torch.bfloat16, device="cuda")
        for _ in range(2):  # (the second layer of a step takes the first one's plan)
            impl.forward(None, q, k, v, kv, md, out)
        torch.cuda.synchronize()
        assert bool((out[T:] == 9.0).all())
        outs.append(out[:T].float())
    assert len(md.plans) == 1 and all(int(e) == 0 for e in impl._error.values())
    assert (outs[0] - outs[1]).abs().max().item() <= 2.0 ** -8 * (6.0 + 6.0) + 2.0 ** -8 * 6.0


def test_backend_cascade_matches_per_request_decode(cuda, monkeypatch):
    vllm = pytest.importorskip("vllm")  # noqa: F841
    import torch
    from spark_b200.plugin.attention import PAGED_ENV, SparkAttentionImpl
    nq, nkv, D, bs, prefix, own = 32, 8, 128, 128, 512, [1, 130, 40, 7, 300]
    g = torch.Generator(device="cuda").manual_seed(4)
    sp, need = prefix // bs, [-(-n // bs) for n in own]
    kv0 = torch.randn((2, sp + sum(need), nkv, bs, D), generator=g, device="cuda").to(torch.bfloat16)
    table = torch.zeros((5, sp + max(need)), dtype=torch.int32, device="cuda")
    table[:, :sp] = torch.arange(sp, device="cuda")
    at = sp
    for r, n in enumerate(need):
        table[r, sp:sp + n] = torch.arange(at, at + n, device="cuda")
        at += n
    lens = [prefix + n for n in own]
    last = torch.tensor(lens, device="cuda") - 1
    slots = table[torch.arange(5, device="cuda"), last // bs].long() * bs + last % bs
    q, k, v = (torch.randn((5, h * D), generator=g, device="cuda").to(torch.bfloat16) for h in (nq, nkv, nkv))
    outs = []
    for on in ("0", "1"):
        monkeypatch.setenv(PAGED_ENV, on)
        impl = SparkAttentionImpl(nq, D, 1 / math.sqrt(D), nkv)
        md = _metadata(lens, [1] * 5, table, slots, prefix)
        out = torch.zeros((5, nq * D), dtype=torch.bfloat16, device="cuda")
        impl.forward(None, q, k, v, kv0.clone(), md, out)
        torch.cuda.synchronize()
        outs.append(out.float())
    assert [p.kind for p in md.plans.values()] == ["prefix"] and all(int(e) == 0 for e in impl._error.values())
    assert (outs[0] - outs[1]).abs().max().item() <= 2.0 ** -8 * (6.0 + 6.0) + 2.0 ** -8 * 6.0
