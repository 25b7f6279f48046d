"""CPU checks of the paged-batch wrappers: sizes that the 32-bit C interface cannot hold are
refused instead of passed on with their upper bits missing."""
from __future__ import annotations

import pytest


@pytest.mark.parametrize("change", [dict(max_tokens=(1 << 32) + 64), dict(max_reqs=(1 << 32) + 4),
                                    dict(nq=(1 << 32) + 8), dict(nkv=(1 << 32) + 2), dict(head_dim=(1 << 32) + 128),
                                    dict(window=(1 << 32) + 8), dict(window=1 << 32), dict(window=1 << 31),
                                    dict(window=-1)])
def test_attn_plan_refuses_sizes_past_32_bits(change):
    import spark_b200
    from spark_b200 import ops
    spark_b200.ensure_built()
    args = {**dict(max_tokens=64, max_reqs=4, nq=8, nkv=2, head_dim=128, device="cuda:0", window=0), **change}
    with pytest.raises(ValueError, match="below 2\\^31"):  # (before anything is allocated)
        ops.AttnPlan(**args)


@pytest.mark.parametrize("what", ["rows", "block_size", "free"])
def test_paged_plan_refuses_sizes_past_32_bits(monkeypatch, what):
    """(on the meta device, where 2^32 rows take no memory; the device checks are stood in for)"""
    import torch
    from spark_b200 import ops
    z = lambda n, t=torch.int32: torch.zeros(n, dtype=t, device="meta")  # noqa: E731
    monkeypatch.setattr(ops, "_home", lambda *a: 0)
    monkeypatch.setattr(ops, "_need_all", lambda *a: None)
    monkeypatch.setattr(ops, "_block_table", lambda *a: None)
    monkeypatch.setattr(ops, "_launch", lambda *a: pytest.fail("launched"))
    rows = (1 << 32) + 5 if what == "rows" else 5
    free = z((1 << 32) + 5) if what == "free" else z(5)
    with pytest.raises(ValueError, match="below 2\\^31"):
        ops.paged_plan_out(z(2), z(2), z((2, 4)), (1 << 32) + 16 if what == "block_size" else 16, z(3), z(2),
                           z(rows, torch.int64), z(rows, torch.int64), z(1), z(1), free_blocks=free, free_head=z(1))


def test_attn_paged_bounded_refuses_a_table_without_rows():
    import ctypes
    import spark_b200
    from spark_b200 import _lib
    spark_b200.ensure_built()
    at, scale = ctypes.c_void_p(0x1000), ctypes.c_float(0.1)  # (never dereferenced)
    for rows in (0, -1):
        assert _lib.lib().spark_attn_paged_bounded(at, 1024, 128, 10, at, at, 4, 16, at, 8, 8, rows, 64, 4, 8, 2, 128, 0,
                                                   scale, at, at, at, at, 1024, 128, at, -1, None) == 2
