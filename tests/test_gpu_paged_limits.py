"""GPU checks of the paged-batch operators at the ends of their ranges: the most rows, plans
and calls that do not belong together, tensors that overlap."""
from __future__ import annotations

import pytest

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
