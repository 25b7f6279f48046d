"""GPU checks of the vLLM backend's paged path against attention in 64 bits on the host,
element by element: u (sum p |v| + |o|) + 2^-12 sum p |v| with u = 2^-8 (the roundings of
the probabilities and of the output; fp32 scores and exponentials), the bound of
test_gpu_paged.  The same bound on oracles with a planted mistake (a length one short, a start one
late, a prefix that is another request's) has to fail: random keys average out, so an absolute bound
would let those pass."""
from __future__ import annotations

import math

import pytest

pytest.importorskip("vllm")
pytestmark = pytest.mark.gpu

U = 2.0 ** -8


def _oracle(q, kv, table, seq_lens, query_lens, nq, nkv, D, window, starts=None, prefix_from=None, prefix=0):
    """float64 outputs and sum p |v| on the host.  ``starts``: where each request's query rows
    begin (default: one behind the other); ``prefix_from``: the request whose pages hold the
    first ``prefix`` positions."""
    import torch
    k, v = kv[0].double(), kv[1].double()  # [pages, nkv, 128, D]
    T, out0 = q.shape[0], 0
    out = torch.zeros((T, nq, D), dtype=torch.float64)
    mag = torch.zeros_like(out)
    for r, (m, n) in enumerate(zip(seq_lens, query_lens)):
        at = torch.arange(m)
        pages = table[r, at // 128].long()
        if prefix_from is not None:
            pages = torch.where(at < prefix, table[prefix_from, at // 128].long(), pages)
        keys, vals = k[pages, :, at % 128], v[pages, :, at % 128]  # [m, nkv, D]
        q0 = out0 if starts is None else starts[r]
        qr = q[q0:q0 + n].double().view(-1, nkv, nq // nkv, D)
        s = torch.einsum("ihgd,jhd->hgij", qr, keys) / math.sqrt(D)
        behind = (m - n + torch.arange(qr.shape[0]))[:, None] - at[None, :]
        hidden = (behind < 0) | (behind >= window) if window else behind < 0
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1).nan_to_num()
        rows = slice(out0, out0 + qr.shape[0])
        out[rows] = torch.einsum("hgij,jhd->ihgd", p, vals).reshape(-1, nq, D)
        mag[rows] = torch.einsum("hgij,jhd->ihgd", p, vals.abs()).reshape(-1, nq, D)
        out0 += n
    return out, mag


def _within(got, out, mag) -> bool:
    tol = U * (mag + out.abs()) + 2.0 ** -12 * mag + 1e-30
    return bool(((got.cpu().double() - out).abs() <= tol).all())


def _builder(layers):
    from spark_b200.plugin.attention import SparkAttentionMetadataBuilder as B, choose_splits, split_tokens
    b = B.__new__(B)
    b.splits, b.layer_names = choose_splits(4096), [f"layer{i}" for i in range(layers)]
    b.max_split_tokens = split_tokens(4096, b.splits)
    return b


def _build(builder, seq_lens, query_lens, table, slots, prefix=0):
    import torch
    from vllm.v1.attention.backend import CommonAttentionMetadata
    start = torch.tensor([0, *torch.tensor(query_lens).cumsum(0).tolist()], dtype=torch.int32)
    return builder.build(prefix, CommonAttentionMetadata(
        query_start_loc=start.cuda(), query_start_loc_cpu=start,
        seq_lens=torch.tensor(seq_lens, dtype=torch.int32, device="cuda"), num_reqs=len(seq_lens),
        num_actual_tokens=int(start[-1]), max_query_len=max(query_lens), max_seq_len=max(seq_lens),
        block_table_tensor=table, slot_mapping=slots))


def _mixed(seq_lens, query_lens, nq, nkv, D, seed):
    """q, k, v rows, a cache that holds the context, the table and the new rows' slots."""
    import torch
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    need = [-(-n // 128) for n in seq_lens]
    perm = torch.randperm(sum(need) + 2, generator=g).to(torch.int32)
    table, at, slots = torch.zeros((len(need), max(need)), dtype=torch.int32), 0, []
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
        p = torch.arange(seq_lens[r] - query_lens[r], seq_lens[r])
        slots.append(table[r, p // 128].long() * 128 + p % 128)
    T = sum(query_lens)
    return (rn(T, nq * D), rn(T, nkv * D), rn(T, nkv * D), rn(2, sum(need) + 2, nkv, 128, D), table.cuda(),
            torch.cat(slots).cuda())


@pytest.mark.parametrize("on", ["0", "1"])
@pytest.mark.parametrize("nq,nkv,D,window", [(32, 8, 128, None), (16, 4, 256, None), (16, 4, 256, 64)])
def test_backend_mixed_batch_matches_float64(cuda, monkeypatch, nq, nkv, D, window, on):
    """A prompt, a chunk and a single token through the torch path and the paged path."""
    import torch
    from spark_b200.plugin.attention import PAGED_ENV, SparkAttentionImpl
    monkeypatch.setenv(PAGED_ENV, on)
    seq_lens, query_lens = [200, 700, 333], [200, 60, 1]
    q, k, v, kv, table, slots = _mixed(seq_lens, query_lens, nq, nkv, D, seed=3)
    impl = SparkAttentionImpl(nq, D, 1 / math.sqrt(D), nkv, sliding_window=window)
    md = _build(_builder(1), seq_lens, query_lens, table, slots)
    out = torch.full((266, nq * D), 9.0, dtype=torch.bfloat16, device="cuda")
    impl.forward(None, q, k, v, kv, md, out)
    torch.cuda.synchronize()
    assert bool((out[261:] == 9.0).all())
    got = out[:261].view(-1, nq, D)
    args = (q.cpu().view(-1, nq, D), kv.cpu(), table.cpu())  # (the new keys are in the cache now)
    rest = (nq, nkv, D, impl.window)
    assert _within(got, *_oracle(*args, seq_lens, query_lens, *rest))
    # planted in the oracle
    for lens in ([199, 700, 333], [200, 699, 333], [200, 700, 332]):
        assert not _within(got, *_oracle(*args, lens, query_lens, *rest)), lens
    assert not _within(got, *_oracle(*args, seq_lens, query_lens, *rest, starts=[0, 199, 260]))
    assert not _within(got, *_oracle(*args, seq_lens, query_lens, *rest, starts=[0, 200, 259]))
    if window:
        assert not _within(got, *_oracle(*args, seq_lens, query_lens, nq, nkv, D, impl.window - 1))


@pytest.mark.parametrize("on", ["0", "1"])
def test_backend_cascade_matches_float64(cuda, monkeypatch, on):
    import torch
    from spark_b200.plugin.attention import PAGED_ENV, SparkAttentionImpl
    monkeypatch.setenv(PAGED_ENV, on)
    nq, nkv, D, prefix, own = 32, 8, 128, 512, [1, 130, 40, 7, 300]
    lens, ones = [prefix + n for n in own], [1] * 5
    q, k, v, kv, table, slots = _mixed(lens, ones, nq, nkv, D, seed=4)
    table[:, :4] = table[:1, :4]
    impl = SparkAttentionImpl(nq, D, 1 / math.sqrt(D), nkv)
    md = _build(_builder(1), lens, ones, table, slots, prefix)
    out = torch.zeros((5, nq * D), dtype=torch.bfloat16, device="cuda")
    impl.forward(None, q, k, v, kv, md, out)
    torch.cuda.synchronize()
    got = out.view(-1, nq, D)
    args, rest = (q.cpu().view(-1, nq, D), kv.cpu(), table.cpu()), (nq, nkv, D, 0)
    assert _within(got, *_oracle(*args, lens, ones, *rest))
    assert (on == "1") == any(p.kind == "prefix" for p in md.plans.values())
    for r in range(5):  # planted in the oracle: a length one short, the prefix a page longer
        assert not _within(got, *_oracle(*args, [n - (i == r) for i, n in enumerate(lens)], ones, *rest)), r
    wide = torch.nn.functional.pad(table.cpu(), (0, 1))
    assert not _within(got, *_oracle(q.cpu().view(-1, nq, D), kv.cpu(), wide, lens, ones, *rest, prefix_from=1,
                                     prefix=prefix + 128))


def test_backend_micro_batches_take_turns(cuda, monkeypatch):
    """Two batches built by one builder whose layers take turns, as micro-batches do."""
    import torch
    from spark_b200.plugin.attention import PAGED_ENV, SparkAttentionImpl
    monkeypatch.setenv(PAGED_ENV, "1")
    nq, nkv, D = 8, 2, 128
    impl, builder, jobs = SparkAttentionImpl(nq, D, 1 / math.sqrt(D), nkv), _builder(2), []
    for seed, (lens, new) in enumerate([([200, 90], [200, 30]), ([150, 260], [1, 9])]):
        q, k, v, kv, table, slots = _mixed(lens, new, nq, nkv, D, seed=seed)
        md = _build(builder, lens, new, table, slots)
        jobs.append((q, k, v, kv, table, lens, new, md, []))
    for _ in range(2):
        for q, k, v, kv, table, lens, new, md, outs in jobs:
            outs.append(torch.zeros_like(q))
            impl.forward(None, q, k, v, kv, md, outs[-1])
    torch.cuda.synchronize()
    for q, k, v, kv, table, lens, new, md, outs in jobs:
        want = _oracle(q.cpu().view(-1, nq, D), kv.cpu(), table.cpu(), lens, new, nq, nkv, D, 0)
        for out in outs:
            assert _within(out.view(-1, nq, D), *want)


def test_backend_raises_a_bad_page_when_the_next_step_is_built(cuda, monkeypatch):
    """A table entry outside the cache: no step is waited for, the next one's metadata raises;
    afterwards the backend goes on, and right."""
    import torch
    from spark_b200.plugin import attention as A
    monkeypatch.setenv(A.PAGED_ENV, "1")
    A.raise_on_error()  # (nothing is left from before)
    nq, nkv, D, lens, new = 8, 2, 128, [200, 90], [200, 30]
    impl, builder = A.SparkAttentionImpl(nq, D, 1 / math.sqrt(D), nkv), _builder(1)
    q, k, v, kv, table, slots = _mixed(lens, new, nq, nkv, D, seed=9)
    bad = table.clone()
    bad[1, 0] = 1 << 20
    impl.forward(None, q, k, v, kv, _build(builder, lens, new, bad, slots), torch.zeros_like(q))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="status 64"):
        _build(builder, lens, new, table, slots)
    out = torch.zeros_like(q)
    impl.forward(None, q, k, v, kv, _build(builder, lens, new, table, slots), out)
    A.raise_on_error()
    assert _within(out.view(-1, nq, D), *_oracle(q.cpu().view(-1, nq, D), kv.cpu(), table.cpu(), lens, new, nq, nkv, D, 0))
    impl.forward(None, q, k, v, kv, _build(builder, lens, new, bad, slots), out)
    with pytest.raises(RuntimeError, match="status 64"):
        A.raise_on_error()


def test_backend_profiling_run_counts_the_workspace(cuda, monkeypatch):
    """The plan of the profiling run is the steps' one: no memory of its size is taken later, also
    when they run on another stream."""
    import torch
    from spark_b200.plugin import attention as A
    monkeypatch.setenv(A.PAGED_ENV, "1")
    monkeypatch.setattr(A, "_pool", A.PlanPool())
    nq, nkv, D, lens, new = 32, 8, 128, [200, 90], [200, 30]
    impl, builder = A.SparkAttentionImpl(nq, D, 1 / math.sqrt(D), nkv), _builder(1)
    q, k, v, kv, table, slots = _mixed(lens, new, nq, nkv, D, seed=10)
    md, out, side = _build(builder, lens, new, table, slots), torch.zeros_like(q), torch.cuda.Stream()
    before = torch.cuda.memory_allocated()  # (with the step's own output, 230 x 4096 x 2 bytes)
    impl.forward(None, torch.zeros((1024, nq * D), dtype=torch.bfloat16, device="cuda"), None, None, None, None,
                 torch.empty_like(q))
    held = torch.cuda.memory_allocated() - before
    assert held > 100 << 20
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        impl.forward(None, q, k, v, kv, md, out)
        A.raise_on_error()
    assert torch.cuda.memory_allocated() - before < held + (1 << 20)
    assert _within(out.view(-1, nq, D), *_oracle(q.cpu().view(-1, nq, D), kv.cpu(), table.cpu(), lens, new, nq, nkv, D, 0))
