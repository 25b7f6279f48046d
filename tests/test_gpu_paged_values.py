"""GPU checks of the paged attention where values or limits are extreme: scores that are not
finite, windows near 2^31, prefixes longer than every request.  Tolerances are those of
test_gpu_paged (bf16 roundings of the probabilities and of the output)."""
from __future__ import annotations

import pytest

from test_gpu_paged import _attn_ref, _batch, _close

pytestmark = pytest.mark.gpu


def _set_key(b, r, pos, value):
    """All kv heads' K of position ``pos`` of request ``r``."""
    page = int(b["table"][r, pos // b["bs"]])
    b["kc"][page, :, pos % b["bs"]] = value


@pytest.mark.parametrize("D,nq,nkv", [(128, 8, 2), (256, 8, 2)])
@pytest.mark.parametrize("new", [300, 1])
def test_attn_prompt_nan_key_reaches_every_row_that_sees_it(cuda, D, nq, nkv, new):
    """Request i holds NaN at key 48 + i (one of each sixteen columns, in a tile that late
    rows see whole): rows at or behind it are NaN throughout, rows in front of it are right."""
    import torch
    from spark_b200 import ops
    ctx = 0 if new > 1 else 299
    b = _batch([ctx] * 16, [new] * 16, nq, nkv, D, 16, seed=60)
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    for i in range(16):
        _set_key(b, i, 48 + i, float("nan"))
    plan = ops.AttnPlan(b["q"].shape[0], 16, nq, nkv, D).update(b["start"], b["lens"])
    out = torch.zeros_like(b["q"])
    ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    assert int(b["err"]) == 0
    for i in range(16):
        first = i * new + max(0, 48 + i - ctx)
        _close(out[i * new:first], ref[i * new:first], mag[i * new:first])
        assert bool(out[first:(i + 1) * new].isnan().all()), i


@pytest.mark.parametrize("D,nq,nkv", [(128, 8, 2), (256, 8, 2)])
@pytest.mark.parametrize("new", [300, 1])
def test_attn_prompt_infinite_scores(cuda, D, nq, nkv, new):
    """A score of +inf makes a row NaN (inf - inf), at each of sixteen columns; one of -inf
    has the weight 0: as if the key were not there."""
    import torch
    from spark_b200 import ops
    ctx = 0 if new > 1 else 299
    b = _batch([ctx] * 16, [new] * 16, nq, nkv, D, 16, seed=61)
    b["q"].copy_(b["q"].abs() + 0.125)  # (positive throughout: q . inf is inf, not NaN)
    plan = ops.AttnPlan(b["q"].shape[0], 16, nq, nkv, D).update(b["start"], b["lens"])
    plain, _ = _attn_ref(b, nq, nkv, D, D ** -0.5)
    for sign in (1.0, -1.0):
        for i in range(16):
            _set_key(b, i, 48 + i, sign * float("inf"))
        out = torch.zeros_like(b["q"])
        ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
        torch.cuda.synchronize()
        assert int(b["err"]) == 0
        ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)  # (softmax: exp(-inf) = 0)
        for i in range(16):
            first, end = i * new + max(0, 48 + i - ctx), (i + 1) * new
            _close(out[i * new:first], ref[i * new:first], mag[i * new:first])
            if sign > 0:
                assert bool(out[first:end].isnan().all()), i
            else:
                _close(out[first:end], ref[first:end], mag[first:end])


@pytest.mark.parametrize("D,nq,nkv", [(128, 8, 2), (256, 8, 2)])
@pytest.mark.parametrize("window", [0x7fffffff, 0x7fff0000, 1 << 30, 0])
def test_attn_prompt_window_larger_than_any_request(cuda, D, nq, nkv, window):
    """A window past every length is no window, also for rows in front of the first key (more
    queries than keys)."""
    import torch
    from spark_b200 import ops
    b = _batch([0, 0], [140, 20], nq, nkv, D, 16, seed=62)
    lens = [100, 20]
    b["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
    b["len"] = lens
    plan = ops.AttnPlan(160, 2, nq, nkv, D, window=window).update(b["start"], b["lens"])
    out = torch.full_like(b["q"], float("nan"))
    ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    assert int(b["err"]) == 0 and int(plan.error) == 0
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    assert bool((out[:40] == 0).all()) and bool((out[40:140] != 0).any())
    _close(out, ref, mag)


@pytest.mark.parametrize("D,nq,nkv", [(128, 8, 2), (256, 8, 2)])
def test_attn_shared_prefix_longer_than_every_request(cuda, D, nq, nkv):
    """A prefix length past all requests (a batch of padded slots in the extreme) reads no
    position that none of them holds: no page id behind their ends is looked at, and what the last
    page carries there does not matter."""
    import torch
    from spark_b200 import ops
    b = _batch([89, 69, 0], [1, 1, 1], nq, nkv, D, 16, seed=63, shared=64)
    prefix = torch.tensor([400], dtype=torch.int32, device="cuda")
    b["table"][1:, :6] = b["table"][0, :6]  # (the longest request holds what all share)
    for lens in ([90, 70, 0], [0, 0, 0]):
        b["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        b["len"] = lens
        plan = ops.AttnPlan(3, 3, nq, nkv, D).update_prefix(b["lens"], prefix)
        out = torch.full_like(b["q"], float("nan"))
        ops.attn_shared_prefix_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
        torch.cuda.synchronize()
        assert int(b["err"]) == 0 and int(plan.error) == 0, lens
        ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
        _close(out, ref, mag)
