"""CPU checks of the vLLM backend's paged path: which plan a step's layers use, what happens to
status words, what the profiling run sets aside.  Plans are stood in for by objects that keep
what they were given; no kernel is launched."""
from __future__ import annotations

import gc

import pytest

pytest.importorskip("vllm")


class FakePlan:
    made: list = []

    def __init__(self, max_tokens, max_reqs, nq, nkv, head_dim, device, window=0):
        import torch
        self.max_tokens, self.max_reqs, self.nq, self.nkv = max_tokens, max_reqs, nq, nkv
        self.head_dim, self.device, self.window = head_dim, device, window
        self.error, self.kind, self.list = torch.zeros(1, dtype=torch.int32), None, None
        FakePlan.made.append(self)

    def update(self, query_start, seq_lens):
        self.kind, self.list = "prompt", seq_lens.tolist()
        return self

    def update_prefix(self, seq_lens, prefix_len):
        self.kind, self.list = "prefix", [int(prefix_len), *seq_lens.tolist()]
        return self


@pytest.fixture
def attention(monkeypatch):
    """The backend's module with fake plans, a pool of its own and the paged path switched on;
    ``seen`` holds the work list of each attention call at the time of the call."""
    from spark_b200.plugin import attention as A
    monkeypatch.setenv(A.PAGED_ENV, "1")
    monkeypatch.setattr(FakePlan, "made", [])
    monkeypatch.setattr(A, "_pool", A.PlanPool())
    monkeypatch.setattr(A.ops, "AttnPlan", FakePlan)
    monkeypatch.setattr(A.ops, "kv_store_", lambda *a: None)
    A.seen = []
    call = lambda q, k, v, table, plan, scale, out, err: A.seen.append((plan.kind, plan.list))  # noqa: E731
    monkeypatch.setattr(A.ops, "attn_prompt_out", call)
    monkeypatch.setattr(A.ops, "attn_shared_prefix_out", call)
    yield A
    del A.seen


def _metadata(A, seq_lens, query_lens, builder=None, prefix=0):
    import torch
    from vllm.v1.attention.backend import CommonAttentionMetadata
    start = torch.tensor([0, *torch.tensor(query_lens).cumsum(0).tolist()], dtype=torch.int32)
    builder = builder or _builder(A)
    return builder.build(prefix, CommonAttentionMetadata(
        query_start_loc=start, query_start_loc_cpu=start, seq_lens=torch.tensor(seq_lens, dtype=torch.int32),
        num_reqs=len(seq_lens), num_actual_tokens=int(start[-1]), max_query_len=max(query_lens),
        max_seq_len=max(seq_lens), block_table_tensor=torch.zeros((len(seq_lens), 8), dtype=torch.int32),
        slot_mapping=torch.zeros(int(start[-1]), dtype=torch.int64)))


def _builder(A, layers=0):
    """A builder without vLLM's configuration, for ``layers`` layers."""
    b = A.SparkAttentionMetadataBuilder.__new__(A.SparkAttentionMetadataBuilder)
    b.splits, b.max_split_tokens, b.layer_names = 16, 128, [f"layer{i}" for i in range(layers)]
    return b


def _layer(impl, md, nq=8, nkv=2, d=128):
    import torch
    t = md.num_actual_tokens
    x = lambda h: torch.zeros((t, h * d), dtype=torch.bfloat16)  # noqa: E731
    return impl.forward(None, x(nq), x(nkv), x(nkv), torch.zeros((2, 1, nkv, 128, d), dtype=torch.bfloat16), md, x(nq))


def test_metadata_alive_together_has_a_plan_each(attention):
    """Two micro-batches whose layers take turns: every call has its own batch's work list."""
    A = attention
    impl = A.SparkAttentionImpl(8, 128, 0.1, 2)
    builder = _builder(A)
    one, two = _metadata(A, [70, 9], [60, 9], builder), _metadata(A, [5, 300], [5, 1], builder)
    for _ in range(2):
        _layer(impl, one)
        _layer(impl, two)
    assert A.seen == [("prompt", [70, 9]), ("prompt", [5, 300])] * 2
    assert len(FakePlan.made) == 2


def test_plans_are_used_again_by_later_steps(attention):
    A = attention
    impl = A.SparkAttentionImpl(8, 128, 0.1, 2)
    for n in (70, 64, 3, 2):
        md = _metadata(A, [n, 9], [n, 9])
        _layer(impl, md)
        _layer(impl, md)
        del md
        gc.collect()
    assert [p.max_tokens for p in FakePlan.made] == [128]


def test_a_larger_step_replaces_the_plan(attention):
    A = attention
    impl = A.SparkAttentionImpl(8, 128, 0.1, 2)
    for n, reqs in ((2, 80), (500, 1), (20, 3), (2, 80)):
        md = _metadata(A, [n] * reqs, [n] * reqs)
        _layer(impl, md)
        del md
        gc.collect()
    assert [(p.max_tokens, p.max_reqs) for p in FakePlan.made] == [(256, 128), (512, 128)]
    assert sum(len(e) for e in A._pool._plans.values()) == 1


def test_layouts_and_windows_have_plans_of_their_own(attention):
    A = attention
    md = _metadata(A, [30], [30])
    full, slide = A.SparkAttentionImpl(16, 256, 0.1, 4), A.SparkAttentionImpl(16, 256, 0.1, 4, sliding_window=16)
    for impl in (full, slide, full):
        _layer(impl, md, 16, 4, 256)
    assert [p.window for p in FakePlan.made] == [0, 17] and len(md.plans) == 2


def _failing(A, monkeypatch, bits):
    """Attention calls set ``bits`` in the word that they are given."""
    monkeypatch.setattr(A.ops, "attn_prompt_out", lambda q, k, v, t, plan, s, out, err: err.bitwise_or_(bits))


@pytest.mark.parametrize("layers", [2, 0])  # (0: a builder that does not know its layers)
def test_status_of_a_step_is_raised_when_a_later_one_is_built(attention, monkeypatch, layers):
    A = attention
    impl, builder = A.SparkAttentionImpl(8, 128, 0.1, 2), _builder(A, layers)
    _failing(A, monkeypatch, 64)
    md = _metadata(A, [30], [30], builder)
    _layer(impl, md)
    _layer(impl, md)
    if not layers:  # (its copy is sent for by the next step's metadata)
        md = _metadata(A, [30], [30], builder)
    with pytest.raises(RuntimeError, match="status 64"):
        _metadata(A, [30], [30], builder)
    _metadata(A, [30], [30], builder)  # raised once; the word starts again from 0
    _failing(A, monkeypatch, 0)
    _layer(impl, md)
    A.raise_on_error()


def test_status_of_the_work_list_is_raised_too(attention):
    A = attention
    impl, builder = A.SparkAttentionImpl(8, 128, 0.1, 2), _builder(A, 1)
    md = _metadata(A, [30], [30], builder)
    _layer(impl, md)
    next(iter(md.plans.values())).error.bitwise_or_(4)  # (what AttnPlan.update reports into)
    _layer(impl, md)
    with pytest.raises(RuntimeError, match="status 4"):
        A.raise_on_error()
    A.raise_on_error()


def test_a_copy_that_is_under_way_is_not_overtaken(attention):
    """Steps built before the last one's copy has arrived: it is raised by the first step that
    finds it there."""
    A = attention

    class Event:
        done = False
        query = lambda self: Event.done  # noqa: E731
        record = synchronize = lambda self: None  # noqa: E731

    status = A._pool.status("cpu")
    status.word.fill_(64)
    status.used()
    status.post()
    status._event = Event()  # (the copy under way)
    for _ in range(3):
        status._used = True
        A._pool.check()
        assert status._posted and status._used
    Event.done = True
    with pytest.raises(RuntimeError):
        A._pool.check()


def test_the_profiling_run_sets_the_workspace_aside(attention, monkeypatch):
    """A run without metadata (vLLM measures its memory) makes a plan per layout for the tokens
    that it carries and the scheduler's requests; the steps use it."""
    import types
    import torch
    A = attention
    config = types.SimpleNamespace(scheduler_config=types.SimpleNamespace(max_num_seqs=200))
    monkeypatch.setattr(A, "get_current_vllm_config_or_none", lambda: config)
    impls = [A.SparkAttentionImpl(16, 256, 0.1, 4, sliding_window=w) for w in (None, 16, 16)]
    x = torch.ones((5000, 16 * 256), dtype=torch.bfloat16)
    for impl in impls:
        assert not impl.forward(None, x, None, None, None, None, x.clone()).any()
    assert [(p.max_tokens, p.max_reqs, p.window) for p in FakePlan.made] == [(8192, 256, 0), (8192, 256, 17)]
    for n in (30, 4000):
        md = _metadata(A, [n] * 3, [n // 3] * 3)
        for impl in impls:
            _layer(impl, md, 16, 4, 256)
        del md
        gc.collect()
    assert len(FakePlan.made) == 2
    assert all(p.error is A._pool.status("cpu").word for p in FakePlan.made)


def test_the_profiling_run_takes_nothing_with_the_switch_off(attention, monkeypatch):
    import torch
    A = attention
    monkeypatch.delenv(A.PAGED_ENV)
    x = torch.ones((50, 8 * 128), dtype=torch.bfloat16)
    A.SparkAttentionImpl(8, 128, 0.1, 2).forward(None, x, None, None, None, None, x)
    assert not FakePlan.made


def test_threads_that_ask_at_once_get_a_plan_each(attention, monkeypatch):
    """Micro-batches may run in threads of their own: a switch between the look at a free plan
    and taking it (here while its size is read) hands it out once."""
    import threading
    import time
    A = attention

    class Slow(FakePlan):
        max_tokens = property(lambda self: (time.sleep(0.05), self._n)[1],
                              lambda self, n: setattr(self, "_n", n))

    monkeypatch.setattr(A.ops, "AttnPlan", Slow)
    layout, mds, got = (8, 2, 128, 0), [_metadata(A, [30], [30]) for _ in range(2)], [None, None]
    A._pool.reserve(layout, "cpu", 64, 4)

    def ask(i):
        got[i] = A._pool.take(layout, "cpu", 30, 1, mds[i])

    threads = [threading.Thread(target=ask, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got[0] is not got[1] and None not in got
