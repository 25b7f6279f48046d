"""GPU checks of the paged-batch operators at the ends of their ranges: the most rows, plans
and calls that do not belong together, tensors that overlap."""
from __future__ import annotations

import pytest

from test_gpu_paged import _attn_ref, _batch, _close

pytestmark = pytest.mark.gpu


def test_paged_plan_of_the_most_rows(cuda):
    """2^31 - 1 rows (32 GB of positions and slots): the rows behind the tokens are 0 and -1 to
    the last, nothing in front of the buffers is written."""
    import torch
    from spark_b200 import ops
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB of free memory")
    i32, rows, guard = {"dtype": torch.int32, "device": "cuda"}, (1 << 31) - 1, 1 << 18
    both = [torch.full((guard + rows,), 77, dtype=torch.int64, device="cuda") for _ in range(2)]
    pos, slots = (t[guard:] for t in both)
    ctx, new = torch.tensor([5, 0], **i32), torch.tensor([3, 2], **i32)
    start, lens, counter, err = (torch.zeros(n, **i32) for n in (3, 2, 1, 1))
    ops.paged_plan_out(ctx, new, torch.tensor([[4], [9]], **i32), 16, start, lens, pos, slots, counter, err)
    torch.cuda.synchronize()
    assert int(err) == 0 and start.tolist() == [0, 3, 5] and lens.tolist() == [8, 2]
    assert pos[:7].tolist() == [5, 6, 7, 0, 1, 0, 0] and slots[:6].tolist() == [69, 70, 71, 144, 145, -1]
    assert all(bool((t[:guard] == 77).all()) for t in both)
    for t, want in ((pos, 0), (slots, -1)):
        for part in t[5:].split(1 << 28):
            assert bool((part == want).all())
    del both, pos, slots
    torch.cuda.empty_cache()


@pytest.mark.parametrize("D,nq,nkv", [(128, 8, 2), (256, 8, 2)])
def test_attn_refuses_a_plan_of_another_shape(cuda, D, nq, nkv):
    """The C entry point given a plan made for other maxima, another head layout or window, or
    none: reported, nothing written; with the plan's own it is right."""
    import torch
    from spark_b200 import ops
    from spark_b200._lib import call
    b = _batch([100, 0], [20, 30], nq, nkv, D, 16, seed=70)
    plan = ops.AttnPlan(64, 4, nq, nkv, D, window=40).update(b["start"], b["lens"])
    out = torch.full_like(b["q"], 3.0)

    def run(buf, **change):
        a = {**dict(tokens=64, reqs=4, nq=nq, nkv=nkv, window=40), **change}
        b["err"].zero_()
        call("spark_attn_paged", b["q"].data_ptr(), nq * D, D, 50, b["kc"].data_ptr(), b["vc"].data_ptr(),
             b["kc"].shape[0], 16, b["table"].data_ptr(), b["table"].stride(0), b["table"].shape[1], a["tokens"],
             a["reqs"], a["nq"], a["nkv"], D, a["window"], D ** -0.5, buf.data_ptr(), plan.part_o.data_ptr(),
             plan.part_ml.data_ptr(), out.data_ptr(), nq * D, D, b["err"].data_ptr(), -1,
             torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return int(b["err"])

    for change in (dict(tokens=63), dict(reqs=3), dict(nq=4), dict(nkv=1), dict(window=0), dict(window=41)):
        assert run(plan.buf, **change) == ops.ERR_PLAN, change
        assert bool((out == 3.0).all())
    assert run(torch.zeros_like(plan.buf)) == ops.ERR_PLAN and bool((out == 3.0).all())
    assert run(plan.buf) == 0
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5, 40)
    _close(out, ref, mag)


def test_attn_plans_have_room_for_an_item_per_block():
    """(each block reads its first item before it knows that the plan is one of its shape)"""
    from spark_b200._lib import lib
    for shape in ((1, 1, 4096, 4096, 128), (1, 1, 8, 1, 128), (1, 1, 592, 592, 256)):
        assert lib().spark_attn_plan_bytes(*shape) >= 64 + 148 * 48


@pytest.mark.parametrize("D,nq,nkv", [(128, 8, 2), (256, 8, 2)])
def test_attn_captured_with_fewer_table_rows_than_a_later_plan(cuda, D, nq, nkv):
    """Only the attention is captured, with a table of two rows; the plan is then made for four
    requests.  What lies behind the table is not read (here: the ids of other pages), the
    requests that it holds are right, the rest is reported."""
    import torch
    from spark_b200 import ops
    b = _batch([100, 0, 40, 300], [20, 30, 1, 1], nq, nkv, D, 16, seed=71)
    plan = ops.AttnPlan(52, 4, nq, nkv, D).update(b["start"][:3], b["lens"][:2])
    out = torch.zeros_like(b["q"])
    run = lambda table: ops.attn_prompt_out(b["q"], b["kc"], b["vc"], table, plan, D ** -0.5, out, b["err"])  # noqa: E731
    run(b["table"][:2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(b["table"][:2])
    plan.update(b["start"], b["lens"])
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert int(b["err"]) == ops.ERR_PAGE
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out[:50], ref[:50], mag[:50])
    assert bool((out[50:] == 0).all())  # (V of a page that is not there: zeros)
    b["err"].zero_()
    run(b["table"])  # the whole table: all right
    torch.cuda.synchronize()
    assert int(b["err"]) == 0
    _close(out, ref, mag)


def test_paged_plan_outputs_between_the_table_rows(cuda):
    """What does not overlap is taken: one int32 buffer holds the table's rows and, between them,
    the counter and the status word; the head next to the lengths."""
    import torch
    from spark_b200 import ops
    i32 = {"dtype": torch.int32, "device": "cuda"}
    buf = torch.zeros((3, 8), **i32)
    buf[:, :6] = -1
    ints = torch.zeros(16, **i32)
    ctx, new, head, start, lens = ints[0:3], ints[3:6], ints[6:7], ints[7:11], ints[11:14]
    new.copy_(torch.tensor([20, 1, 3]))
    both = torch.zeros(2 * 26, dtype=torch.int64, device="cuda")
    pos, slots = both[:26], both[26:]
    ops.paged_plan_out(ctx, new, buf[:, :6], 16, start, lens, pos, slots, buf[0, 6:7], buf[1, 7:8],
                       free_blocks=torch.arange(5, 15, **i32), free_head=head)
    torch.cuda.synchronize()
    assert buf.tolist() == [[5, 6, -1, -1, -1, -1, 0, 0], [7, -1, -1, -1, -1, -1, 0, 0], [8, -1, -1, -1, -1, -1, 0, 0]]
    assert int(head) == 4 and start.tolist() == [0, 20, 21, 24] and lens.tolist() == [20, 1, 3]
    assert slots.tolist() == [*range(80, 100), 112, 128, 129, 130, -1, -1]
