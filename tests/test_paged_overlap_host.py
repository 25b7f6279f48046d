"""CPU checks: the paged-batch entry points refuse outputs that overlap their inputs or one
another (other blocks read and write them at the same time).  Addresses are stand-ins and never
dereferenced; nothing is launched by a call that is refused."""
from __future__ import annotations

import ctypes

import pytest

INVALID = 1


@pytest.fixture(scope="module")
def L():
    import spark_b200
    from spark_b200 import _lib

    spark_b200.ensure_built()
    return _lib.lib()


# 4 requests, 9 free ids, 6 rows; every tensor in a page of its own
PLAN = dict(ctx=0x1000, new=0x2000, reqs=4, free=0x3000, num_free=9, head=0x4000, head_out=0x4000, table=0x5000, stride=8,
            width=8, bs=16, rows=6, qs=0x6000, sl=0x7000, pos=0x8000, slots=0x9000, counter=0xa000, error=0xb000,
            stream=None)
ROWS = dict(qkv=0x10000, stride=1536, rows=4, nq=8, nkv=2, D=128, qg=None, kg=None, eps=1e-6, cs=0x20000, max_pos=100,
            rot=128, pos=0x30000, slots=0x31000, bs=16, blocks=4, kc=0x40000, vc=0x60000, q=0x80000, error=0x90000,
            stream=None)


def _call(fn, args):
    return fn(*(ctypes.c_void_p(v) if isinstance(v, int) and v >= 0x1000 else v for v in args.values()))


@pytest.mark.parametrize("change", [
    dict(qs=0x2000 - 16),         # its fifth entry is the first length
    dict(qs=0x1000 + 12), dict(sl=0x2000 + 4), dict(pos=0x1000 - 40), dict(slots=0x2000), dict(table=0x1000 - 4 * 31),
    dict(table=0x3000 + 32), dict(pos=0x3000 - 8), dict(head_out=0x3000 + 4), dict(head_out=0x1000),
    dict(sl=0x6000 + 16), dict(slots=0x8000 + 40), dict(counter=0xb000), dict(error=0x6000), dict(head=0xb000),
    dict(table=0x6000 - 8), dict(counter=0x5000 + 4 * 31),
    dict(stride=10, counter=0x5000 + 4 * 10), dict(stride=10, counter=0x5000 + 4 * 17), dict(stride=10, sl=0x5000 + 32)])
def test_paged_plan_refuses_overlapping_tensors(L, change):
    assert _call(L.spark_paged_plan, {**PLAN, **change}) == INVALID


@pytest.mark.parametrize("change", [
    dict(q=0x10000), dict(q=0x10000 + 2 * (3 * 1536 + 1520)), dict(q=0x10000 - 16), dict(kc=0x10000), dict(vc=0x10000),
    dict(vc=0x40000), dict(vc=0x40000 + 2 * 16368), dict(q=0x40000), dict(q=0x60000 + 2 * 16368),
    dict(rows=1, q=0x10000 + 16)])
def test_rope_store_refuses_overlapping_tensors(L, change):
    assert _call(L.spark_qk_norm_rope_store_rows, {**ROWS, **change}) == INVALID
