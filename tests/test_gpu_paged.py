"""GPU checks of the paged-batch operators: block tables and slot maps (paged_plan_out),
norm + rotation + store (qk_norm_rope_store_rows) and the paged attention (AttnPlan,
attn_prompt_out, attn_shared_prefix_out), each against a plain form in 64 bits.

Tolerances.  u = 2^-8 bounds the relative rounding of one bf16 (eps / 2).
* rotation: fp32 arithmetic (a few 2^-24 relative to the products) and one bf16 rounding:
  |err| <= u |y| + 2^-20 (|a c| + |b s|).
* attention: probabilities are rounded to bf16 before they multiply v, the output once more:
  |err| <= u sum p |v| + u |o|; the scores are fp32 sums of D products (error below
  D 2^-24 sum |q k| scale < 2^-14 here) and the exponential is good to 2^-13, both relative
  errors of p: 2^-12 sum p |v| covers them.
"""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


# ------------------------------------------------------------------ plans
def _plan_ref(ctx, new, table, bs, free, head):
    table = [row[:] for row in table]
    start, pos, slot = [0], [], []
    for r, (c, n) in enumerate(zip(ctx, new)):
        for p in range(-(-c // bs), -(-(c + n) // bs)):
            if free is not None:
                table[r][p] = free[head]
                head += 1
        for x in range(c, c + n):
            pos.append(x)
            slot.append(table[r][x // bs] * bs + x % bs)
        start.append(start[-1] + n)
    return start, pos, slot, table, head


def _plan_call(ctx, new, table, bs, rows, free=None, head=None, in_place=True, extra_cols=0):
    import torch
    from spark_b200 import ops
    i32 = {"dtype": torch.int32, "device": "cuda"}
    R = len(ctx)
    wide = torch.full((R, len(table[0]) + extra_cols), 77, **i32)
    t = wide[:, :len(table[0])]
    t.copy_(torch.tensor(table, **i32))
    o = {"query_start": torch.full((R + 1,), -5, **i32), "seq_lens": torch.full((R,), -5, **i32),
         "positions": torch.full((rows,), -9, dtype=torch.int64, device="cuda"),
         "slot_mapping": torch.full((rows,), -9, dtype=torch.int64, device="cuda"),
         "counter": torch.zeros(1, **i32), "error": torch.zeros(1, **i32)}
    kw = {}
    if free is not None:
        kw = {"free_blocks": torch.tensor(free, **i32), "free_head": torch.tensor([head], **i32)}
        if not in_place:
            kw["free_head_out"] = torch.full((1,), -3, **i32)
    ops.paged_plan_out(torch.tensor(ctx, **i32), torch.tensor(new, **i32), t, bs, **o, **kw)
    torch.cuda.synchronize()
    o["table"], o["wide"] = t, wide
    o["head"] = kw.get("free_head_out", kw.get("free_head"))
    assert int(o["counter"]) == 0
    return o


PLANS = [  # (cached, new, block size, spare rows)
    ([0], [1], 128, 0),
    ([0], [0], 16, 3),
    ([5, 128, 127, 0, 300], [1, 1, 1, 1, 1], 128, 0),
    ([0, 17, 64, 0, 63, 1000], [130, 0, 64, 0, 2, 1], 16, 61),
    ([0] * 700, [(7 * i) % 31 for i in range(700)], 16, 100),
    ([i * 3 for i in range(1500)], [1] * 1500, 64, 0),
    ([0, 0], [70001, 33], 48, 7),
    ([i % 40 for i in range(8192)], [i % 3 for i in range(8192)], 16, 5),  # the most requests: 98 KB of starts
]


@pytest.mark.parametrize("which", range(len(PLANS)))
@pytest.mark.parametrize("allocate", [True, False])
def test_paged_plan_matches_list_form(cuda, which, allocate):
    import random
    ctx, new, bs, spare = PLANS[which]
    rng = random.Random(which)
    width = max(1, max(-(-(c + n) // bs) for c, n in zip(ctx, new))) + 1
    pages = sum(-(-(c + n) // bs) for c, n in zip(ctx, new)) + 9
    ids = list(range(pages))
    rng.shuffle(ids)
    table = [[-1] * width for _ in ctx]
    for r, (c, n) in enumerate(zip(ctx, new)):
        for p in range(-(-(c if allocate else c + n) // bs)):
            table[r][p] = ids.pop()
    free, head = ([-1, -1] + ids, 2) if allocate else (None, None)
    start, pos, slot, want, head2 = _plan_ref(ctx, new, table, bs, free, head)
    o = _plan_call(ctx, new, table, bs, sum(new) + spare, free, head, in_place=which % 2 == 0, extra_cols=3)
    assert int(o["error"]) == 0
    assert o["query_start"].tolist() == start
    assert o["seq_lens"].tolist() == [c + n for c, n in zip(ctx, new)]
    assert o["positions"].tolist() == pos + [0] * spare
    assert o["slot_mapping"].tolist() == slot + [-1] * spare
    assert o["table"].tolist() == want
    assert bool((o["wide"][:, width:] == 77).all())  # columns behind the table left alone
    if allocate:
        assert int(o["head"]) == head2


@pytest.mark.parametrize("case", ["pages", "width", "rows", "negative", "head"])
def test_paged_plan_that_does_not_fit_takes_nothing(cuda, case):
    from spark_b200 import ops
    ctx, new, bs = [100, 0, 30], [60, 40, 2], 16
    table = [[-1] * 10 for _ in ctx]
    table[0][:7], table[2][:2] = list(range(7)), [7, 8]
    free, head, rows = list(range(9, 30)), 4, 102
    bit = {"pages": ops.ERR_NO_PAGES, "width": ops.ERR_TABLE_WIDTH, "rows": ops.ERR_NO_ROWS,
           "negative": ops.ERR_LENGTH, "head": ops.ERR_NO_PAGES}[case]
    if case == "pages":
        free = free[:8]
    elif case == "width":
        new[0] = 61
    elif case == "rows":
        rows = 101
    elif case == "negative":
        new[1] = -1
    else:
        head = -1
    o = _plan_call(ctx, new, table, bs, rows, free, head)
    assert int(o["error"]) & bit
    assert o["table"].tolist() == table and int(o["head"]) == head
    assert o["query_start"].tolist() == [0] * 4 and o["seq_lens"].tolist() == [0] * 3
    assert bool((o["slot_mapping"] == -1).all()) and bool((o["positions"] == 0).all())


def test_paged_plan_page_without_id_is_reported(cuda):
    from spark_b200 import ops
    o = _plan_call([0], [20], [[3, -1]], 16, 20)
    assert int(o["error"]) == ops.ERR_PAGE
    assert o["slot_mapping"].tolist() == list(range(48, 64)) + [-1] * 4


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("rows,nq,nkv,D,rot,norm,extra", [
    (1, 32, 8, 128, 128, False, 0), (1, 32, 8, 128, 128, True, 0), (77, 7, 1, 128, 64, True, 8),
    (130, 16, 4, 256, 64, True, 16), (33, 6, 2, 256, 256, False, 0), (2049, 5, 5, 128, 16, True, 24),
    (300, 16, 4, 256, 256, True, 0)])
def test_rope_store_matches_float64(cuda, rows, nq, nkv, D, rot, norm, extra):
    import torch
    from spark_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(rows + D + rot)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    cols = (nq + 2 * nkv) * D
    qkv = (rn(rows, cols + extra) * torch.exp(rn(rows, 1))).to(torch.bfloat16)
    bs, max_pos = 16, 5000
    blocks = -(-rows // bs) + 2
    cs = (torch.rand((max_pos, rot), generator=g, device="cuda") * 2 - 1).to(torch.bfloat16)
    pos = torch.randint(0, max_pos, (rows,), generator=g, device="cuda")
    slots = torch.randperm(blocks * bs, generator=g, device="cuda")[:rows].contiguous()
    if rows > 5:
        slots[3] = -1  # a padding row
    kc, vc = rn(blocks, nkv, bs, D).to(torch.bfloat16), rn(blocks, nkv, bs, D).to(torch.bfloat16)
    k0, v0 = kc.clone(), vc.clone()
    qg, kg = ((1 + 0.2 * rn(D)).to(torch.bfloat16), (1 + 0.2 * rn(D)).to(torch.bfloat16)) if norm else (None, None)
    q = torch.full((rows, nq, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.qk_norm_rope_store_rows(qkv, nq, nkv, D, qg, kg, 1e-6, cs, pos, slots, kc, vc, q, err)
    torch.cuda.synchronize()
    assert int(err) == 0
    x = qkv[:, :cols].double().view(rows, nq + 2 * nkv, D)
    y = x[:, :nq + nkv].clone()
    if norm:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)
        y[:, :nq] *= qg.double()
        y[:, nq:] *= kg.double()
    c, s = cs.double()[pos][:, None, :rot // 2], cs.double()[pos][:, None, rot // 2:]
    a, b = y[..., :rot // 2].clone(), y[..., rot // 2:rot].clone()
    y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    noise = torch.cat([a.abs() + b.abs(), a.abs() + b.abs(), y[..., rot:].abs()], -1) * 2.0 ** -20
    tol = U * y.abs() + noise
    assert bool(((q.double() - y[:, :nq]).abs() <= tol[:, :nq]).all())
    live = slots >= 0
    blk, off = slots[live] // bs, slots[live] % bs
    assert bool(((kc[blk, :, off].double() - y[live, nq:]).abs() <= tol[live, nq:]).all())
    assert torch.equal(vc[blk, :, off], qkv[:, :cols].view(rows, -1, D)[live, nq + nkv:])
    kc[blk, :, off], vc[blk, :, off] = k0[blk, :, off], v0[blk, :, off]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)  # nothing else was written


def test_rope_store_without_norm_is_bitwise_the_row_kernel(cuda):
    """Without gammas the rotation is spark_rope_neox_rows' arithmetic."""
    import torch
    from spark_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(9)
    rows, nq, nkv, D, rot = 50, 8, 2, 256, 64
    qkv = torch.randn((rows, (nq + 2 * nkv) * D), generator=g, device="cuda").to(torch.bfloat16)
    cs = (torch.rand((200, rot), generator=g, device="cuda") * 2 - 1).to(torch.bfloat16)
    kc = torch.zeros((1, nkv, 64, D), dtype=torch.bfloat16, device="cuda")
    vc, q = torch.zeros_like(kc), torch.zeros((rows, nq, D), dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    pos = torch.arange(30, 30 + rows, device="cuda")
    ops.qk_norm_rope_store_rows(qkv, nq, nkv, D, None, None, 0.0, cs, pos, torch.arange(rows, device="cuda"), kc, vc,
                                q, err)
    ref = qkv.clone()
    ops.rope_rows_(ref, nq + nkv, D, rot, cs, 30)
    ref = ref.view(rows, -1, D)
    torch.cuda.synchronize()
    assert torch.equal(q, ref[:, :nq]) and torch.equal(kc[0].transpose(0, 1)[:rows], ref[:, nq:nq + nkv])
    assert int(err) == 0


def test_rope_store_reports_positions_and_slots_out_of_range(cuda):
    import torch
    from spark_b200 import ops
    bf = {"dtype": torch.bfloat16, "device": "cuda"}
    qkv = torch.ones((4, 3 * 128), **bf)
    kc, vc, q = torch.zeros((2, 1, 16, 128), **bf), torch.zeros((2, 1, 16, 128), **bf), torch.zeros((4, 1, 128), **bf)
    cs = torch.ones((10, 128), **bf)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 10, -1, 9], device="cuda")
    slots = torch.tensor([0, 1, 2, 1 << 40], device="cuda")
    ops.qk_norm_rope_store_rows(qkv, 1, 1, 128, None, None, 0.0, cs, pos, slots, kc, vc, q, err)
    torch.cuda.synchronize()
    assert int(err) == ops.ERR_POSITION | ops.ERR_SLOT
    assert bool((q[1] == 0).all()) and bool((q[2] == 0).all()) and bool((kc[0, 0, 1:] == 0).all())
    assert bool((vc[0, 0, :3] == 1).all()) and bool((vc.view(-1, 128)[3:] == 0).all())


# ------------------------------------------------------------------ attention
def _batch(ctx, new, nq, nkv, D, bs, seed, shared=0, scale_q=1.0):
    """Random q, caches whose every row that no request holds is NaN, tables whose entries
    behind a request's pages are no page ids."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    lens = [c + n for c, n in zip(ctx, new)]
    need = [-(-m // bs) for m in lens]
    sp = shared // bs
    blocks = sp + sum(max(0, n - sp) for n in need) + 3
    perm = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(ctx), max(need) + 3), 1 << 30, dtype=torch.int32, device="cuda")
    table[:, 1::2] = -7
    kc, vc = rn(blocks, nkv, bs, D), rn(blocks, nkv, bs, D)
    held = torch.zeros((blocks, bs), dtype=torch.bool, device="cuda")
    off = sp
    for r, n in enumerate(need):
        own = max(0, n - sp)
        table[r, :min(n, sp)] = perm[:min(n, sp)]
        table[r, sp:sp + own] = perm[off:off + own]
        off += own
        at = torch.arange(lens[r], device="cuda")
        held[table[r, at // bs].long(), at % bs] = True
    kc.masked_fill_(~held[:, None, :, None], float("nan"))
    vc.masked_fill_(~held[:, None, :, None], float("nan"))
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    i32 = {"dtype": torch.int32, "device": "cuda"}
    q = (torch.randn((start[-1], nq, D), generator=g, device="cuda") * scale_q).to(torch.bfloat16)
    return {"q": q, "kc": kc, "vc": vc, "table": table, "start": torch.tensor(start, **i32),
            "lens": torch.tensor(lens, **i32), "err": torch.zeros(1, **i32), "new": new, "len": lens, "bs": bs}


def _attn_ref(b, nq, nkv, D, scale, window=0):
    """float64 outputs and sum p |v| (the scale of the tolerance)."""
    import torch
    out = torch.zeros(b["q"].shape, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    t0 = 0
    for r, (n, m) in enumerate(zip(b["new"], b["len"])):
        if n == 0:  # (its table may hold no page at all)
            continue
        at = torch.arange(m, device="cuda")
        blk, off = b["table"][r, at // b["bs"]].long(), at % b["bs"]
        pos = m - n + torch.arange(n, device="cuda")
        behind = pos[:, None] - at[None, :]
        masked = (behind < 0) | (behind >= window) if window else behind < 0
        for h in range(nq):
            k, v = b["kc"][blk, h * nkv // nq, off].double(), b["vc"][blk, h * nkv // nq, off].double()
            s = b["q"][t0:t0 + n, h].double() @ k.t() * scale
            s.masked_fill_(masked, float("-inf"))
            p = torch.nan_to_num(torch.softmax(s, -1))  # (a row without keys: zero)
            out[t0:t0 + n, h], mag[t0:t0 + n, h] = p @ v, p @ v.abs()
        t0 += n
    return out, mag


def _close(got, ref, mag):
    err = (got.double() - ref).abs()
    tol = U * (mag + ref.abs()) + 2.0 ** -12 * mag + 1e-30
    bad = ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((err / tol).nan_to_num(1e9).max()))


PROMPTS = [  # (cached, new, nq, nkv, D, block size, window)
    ([0], [1], 32, 8, 128, 128, 0),
    ([0], [2], 8, 8, 128, 16, 0),
    ([0], [128], 4, 1, 128, 128, 0),
    ([0], [129], 32, 8, 128, 128, 0),
    ([0], [1000], 8, 2, 128, 64, 0),
    ([0, 0, 0, 0], [63, 64, 65, 300], 8, 2, 128, 128, 0),
    ([300, 0, 127, 128, 1], [1, 200, 1, 40, 3], 8, 2, 128, 16, 0),
    ([5000], [1], 32, 8, 128, 128, 0),
    ([4999, 0, 250, 1300], [1, 1, 1, 1], 32, 8, 128, 128, 0),
    ([4000], [70], 8, 2, 128, 32, 0),
    ([0, 900], [500, 100], 6, 2, 128, 48, 0),   # three heads per kv head: rows left over in a tile
    ([0, 33], [150, 20], 28, 4, 128, 128, 0),   # seven
    ([10], [90], 40, 1, 128, 16, 0),            # forty
    ([0, 200], [40, 3], 128, 1, 128, 128, 0),   # one token a tile
    ([0, 700], [700, 33], 8, 2, 128, 64, 100),
    ([900, 1500], [1, 1], 8, 2, 128, 16, 17),
    ([1000], [300], 4, 4, 128, 128, 1),         # a window of the token itself
    ([0], [1], 16, 4, 256, 128, 0),
    ([0, 0, 513], [127, 128, 130], 16, 4, 256, 128, 0),
    ([700, 0], [600, 800], 16, 4, 256, 128, 513),
    ([3000, 2999, 10], [1, 1, 1], 16, 4, 256, 64, 0),
    ([3000], [1], 16, 4, 256, 16, 513),
    ([100], [257], 12, 2, 256, 16, 0),
]


@pytest.mark.parametrize("which", range(len(PROMPTS)))
def test_attn_prompt_matches_float64(cuda, which):
    import torch
    from spark_b200 import ops
    ctx, new, nq, nkv, D, bs, window = PROMPTS[which]
    b = _batch(ctx, new, nq, nkv, D, bs, seed=100 + which, scale_q=1.0 + which % 3)
    scale = D ** -0.5
    T = b["q"].shape[0]
    plan = ops.AttnPlan(T + which % 4, len(ctx) + which % 3, nq, nkv, D, window=window)
    plan.update(b["start"], b["lens"])
    out = torch.full_like(b["q"], float("nan"))
    ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, scale, out, b["err"])
    torch.cuda.synchronize()
    assert int(b["err"]) == 0 and int(plan.error) == 0
    ref, mag = _attn_ref(b, nq, nkv, D, scale, window)
    _close(out, ref, mag)


def test_attn_prompt_rows_without_keys_and_behind_the_batch(cuda):
    """More queries than keys (the first rows see nothing: zero), requests without tokens or
    keys, rows behind the last token left as they were."""
    import torch
    from spark_b200 import ops
    nq, nkv, D, bs = 8, 2, 128, 16
    b = _batch([0, 0, 0, 40], [10, 0, 5, 7], nq, nkv, D, bs, seed=3)
    lens = torch.tensor([4, 9, 0, 47], dtype=torch.int32, device="cuda")
    plan = ops.AttnPlan(64, 8, nq, nkv, D)
    plan.update(b["start"], lens)
    q = torch.cat([b["q"], torch.full((6, nq, D), float("nan"), dtype=torch.bfloat16, device="cuda")])
    out = torch.full_like(q, 7.0)
    ops.attn_prompt_out(q, b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    assert int(b["err"]) == 0 and int(plan.error) == 0
    b["len"] = lens.tolist()
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out[:22], ref, mag)
    assert bool((out[:6] == 0).all()) and bool((out[10:15] == 0).all()) and bool((out[22:] == 7.0).all())


def test_attn_prompt_strided_views_and_other_stream(cuda):
    """q a view of a fused qkv output, out a view of a wider buffer whose other columns stay;
    the whole step on a side stream."""
    import torch
    from spark_b200 import ops
    nq, nkv, D, bs = 8, 2, 128, 16
    b = _batch([40, 0], [50, 90], nq, nkv, D, bs, seed=4)
    T = 140
    qkv = torch.randn((T, (nq + 2 * nkv) * D + 24), device="cuda").to(torch.bfloat16)
    q = qkv[:, :nq * D].view(T, nq, D)
    q.copy_(b["q"])
    wide = torch.full((T, nq, D + 8), 3.0, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan = ops.AttnPlan(T, 2, nq, nkv, D)
        plan.update(b["start"], b["lens"])
        ops.attn_prompt_out(q, b["kc"], b["vc"], b["table"], plan, D ** -0.5, wide[..., :D], b["err"])
    side.synchronize()
    assert int(b["err"]) == 0
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(wide[..., :D], ref, mag)
    assert bool((wide[..., D:] == 3.0).all())


def test_attn_prompt_is_deterministic_and_follows_a_captured_plan(cuda):
    """A captured plan + attention replays for other lengths written into the same tensors;
    the same inputs give the same bits each time."""
    import torch
    from spark_b200 import ops
    nq, nkv, D, bs = 32, 8, 128, 128
    b = _batch([3000, 10, 700], [1, 60, 90], nq, nkv, D, bs, seed=5)
    T = b["q"].shape[0]
    plan = ops.AttnPlan(T, 3, nq, nkv, D)
    out = torch.zeros_like(b["q"])

    def step():
        plan.update(b["start"], b["lens"])
        ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])

    step()
    torch.cuda.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), first.view(torch.int16))
    lens = [2500, 65, 400]
    b["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    b["len"] = lens
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out, ref, mag)
    assert int(b["err"]) == 0


def test_attn_prompt_reports_bad_pages_and_starts(cuda):
    import torch
    from spark_b200 import ops
    nq, nkv, D, bs = 8, 2, 128, 16
    b = _batch([0, 100], [30, 20], nq, nkv, D, bs, seed=6)
    good = b["table"].clone()
    plan = ops.AttnPlan(50, 2, nq, nkv, D)
    plan.update(b["start"], b["lens"])
    out = torch.zeros_like(b["q"])
    for bad in (-1, b["kc"].shape[0], 1 << 30):
        b["err"].zero_()
        b["table"].copy_(good)
        b["table"][1, 3] = bad
        ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
        torch.cuda.synchronize()
        assert int(b["err"]) == ops.ERR_PAGE
        b["table"].copy_(good)
        ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
        _close(out[:30], ref[:30], mag[:30])  # the other request is right
    # a table too narrow for the lengths
    b["err"].zero_()
    ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"][:, :5], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    assert int(b["err"]) == ops.ERR_PAGE
    for starts in ([0, 30, 51], [0, -1, 50], [30, 0, 50]):
        plan.error.zero_()
        plan.update(torch.tensor(starts, dtype=torch.int32, device="cuda"), b["lens"])
        b["err"].zero_()
        ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
        torch.cuda.synchronize()
        assert int(plan.error) == ops.ERR_LENGTH and int(b["err"]) == 0


@pytest.mark.parametrize("n", [-1, 0x7fff0001, 0x7fffffff])
def test_attn_plan_lengths_out_of_range(cuda, n):
    """A request of no valid length is left out and reported; the others are right."""
    import torch
    from spark_b200 import ops
    nq, nkv, D, bs = 8, 2, 128, 16
    b = _batch([0, 100], [30, 20], nq, nkv, D, bs, seed=7)
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    b["lens"][1] = n
    plan = ops.AttnPlan(50, 2, nq, nkv, D).update(b["start"], b["lens"])
    out = torch.full_like(b["q"], 3.0)
    ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    assert int(plan.error) == ops.ERR_LENGTH and int(b["err"]) == 0
    _close(out[:30], ref[:30], mag[:30])
    assert bool((out[30:] == 3.0).all())
    # a prefix of no valid length counts as none
    one = _batch([40, 60], [1, 1], nq, nkv, D, bs, seed=8)
    plan = ops.AttnPlan(2, 2, nq, nkv, D).update_prefix(one["lens"], torch.tensor([n], dtype=torch.int32, device="cuda"))
    out = torch.full_like(one["q"], 3.0)
    ops.attn_shared_prefix_out(one["q"], one["kc"], one["vc"], one["table"], plan, D ** -0.5, out, one["err"])
    torch.cuda.synchronize()
    assert int(plan.error) == ops.ERR_LENGTH and int(one["err"]) == 0
    _close(out, *_attn_ref(one, nq, nkv, D, D ** -0.5))


def test_paged_plan_refuses_outputs_that_are_inputs(cuda):
    import torch
    from spark_b200 import ops
    from spark_b200._lib import SparkError
    z = lambda n, t=torch.int32: torch.zeros(n, dtype=t, device="cuda")  # noqa: E731
    ctx = z(2)
    with pytest.raises(SparkError):  # lengths advanced in place: other blocks still read them
        ops.paged_plan_out(ctx, z(2), z((2, 4)), 16, z(3), ctx, z(4, torch.int64), z(4, torch.int64), z(1), z(1))


PREFIXES = [  # (prefix, own tokens of each request, nq, nkv, D, block size)
    (128, [1, 2], 8, 2, 128, 128),
    (2048, [1, 100, 7, 300, 128, 129, 1, 1], 32, 8, 128, 128),
    (256, list(range(1, 38)), 8, 2, 128, 16),
    (1024, [5] * 70, 28, 4, 128, 64),
    (640, [1, 600, 50], 16, 4, 256, 128),
    (48, [3, 1], 6, 2, 256, 16),
    (0, [9, 300], 8, 2, 128, 16),
    (4096, [1], 128, 1, 128, 128),
]


@pytest.mark.parametrize("which", range(len(PREFIXES)))
def test_attn_shared_prefix_matches_float64(cuda, which):
    import torch
    from spark_b200 import ops
    prefix, own, nq, nkv, D, bs = PREFIXES[which]
    b = _batch([prefix + n - 1 for n in own], [1] * len(own), nq, nkv, D, bs, seed=200 + which, shared=prefix,
               scale_q=1.0 + which % 2)
    plan = ops.AttnPlan(len(own), len(own), nq, nkv, D)
    plan.update_prefix(b["lens"], torch.tensor([prefix], dtype=torch.int32, device="cuda"))
    out = torch.full_like(b["q"], float("nan"))
    ops.attn_shared_prefix_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    assert int(b["err"]) == 0 and int(plan.error) == 0
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out, ref, mag)


def test_attn_shared_prefix_padded_batch_and_uneven_prefix(cuda):
    """A prefix that ends inside a page, a padded slot (length 0: zero), a request shorter
    than the prefix."""
    import torch
    from spark_b200 import ops
    nq, nkv, D, bs = 8, 2, 128, 16
    b = _batch([199, 160, 176], [1, 1, 1], nq, nkv, D, bs, seed=8, shared=160)
    lens = torch.tensor([200, 100, 0], dtype=torch.int32, device="cuda")
    plan = ops.AttnPlan(3, 3, nq, nkv, D)
    plan.update_prefix(lens, torch.tensor([155], dtype=torch.int32, device="cuda"))
    out = torch.full_like(b["q"], float("nan"))
    ops.attn_shared_prefix_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    assert int(b["err"]) == 0 and int(plan.error) == 0
    b["len"] = lens.tolist()
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out, ref, mag)
    assert bool((out[2] == 0).all())


def test_paged_operators_run_together_over_steps(cuda):
    """Two packed prompts, then decode steps through plan -> rows -> attention with pages from
    a free list, against float64 attention over the keys gathered from the caches."""
    import torch
    from spark_b200 import ops
    nq, nkv, D, bs, R = 8, 2, 128, 16, 3
    i32, bf = {"dtype": torch.int32, "device": "cuda"}, {"dtype": torch.bfloat16, "device": "cuda"}
    g = torch.Generator(device="cuda").manual_seed(12)
    blocks = 40
    kc, vc = torch.full((blocks, nkv, bs, D), float("nan"), **bf), torch.full((blocks, nkv, bs, D), float("nan"), **bf)
    free = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    head, counter, error = torch.zeros(1, **i32), torch.zeros(1, **i32), torch.zeros(1, **i32)
    table = torch.full((R, 12), -1, **i32)
    ctx = torch.zeros(R, **i32)
    qg, kg = torch.ones(D, **bf), torch.ones(D, **bf)
    cs = (torch.rand((512, D), generator=g, device="cuda") * 2 - 1).to(torch.bfloat16)
    plan = ops.AttnPlan(160, R, nq, nkv, D)
    total = [0] * R
    for new in ([70, 33, 0], [1, 1, 41], [1, 1, 1], [1, 0, 1]):
        rows = sum(new) + 5
        start, lens = torch.zeros(R + 1, **i32), torch.zeros(R, **i32)
        pos = torch.zeros(rows, dtype=torch.int64, device="cuda")
        slots = torch.zeros_like(pos)
        ops.paged_plan_out(ctx, torch.tensor(new, **i32), table, bs, start, lens, pos, slots, counter, error,
                           free_blocks=free, free_head=head)
        plan.update(start, lens)
        qkv = torch.randn((rows, (nq + 2 * nkv) * D), generator=g, device="cuda").to(torch.bfloat16)
        q, out = torch.zeros((rows, nq, D), **bf), torch.full((rows, nq, D), 5.0, **bf)
        ops.qk_norm_rope_store_rows(qkv, nq, nkv, D, qg, kg, 1e-6, cs, pos, slots, kc, vc, q, error)
        ops.attn_prompt_out(q, kc, vc, table, plan, D ** -0.5, out, error)
        torch.cuda.synchronize()
        total = [a + n for a, n in zip(total, new)]
        assert int(error) == 0 and lens.tolist() == total
        b = {"q": q[:sum(new)], "kc": kc, "vc": vc, "table": table, "new": new, "len": total, "bs": bs}
        ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
        _close(out[:sum(new)], ref, mag)
        assert bool((out[sum(new):] == 5.0).all())
        ctx.copy_(lens)
    assert int(head) == sum(-(-t // bs) for t in total)


def test_paged_custom_ops(cuda):
    """torch.ops.spark_b200.attn_prompt / attn_shared_prefix / qk_norm_rope_store_rows."""
    import torch
    from spark_b200 import ops  # noqa: F401
    nq, nkv, D, bs = 8, 2, 128, 16
    b = _batch([31, 0], [20, 9], nq, nkv, D, bs, seed=21)
    out = torch.ops.spark_b200.attn_prompt(b["q"], b["kc"], b["vc"], b["table"], b["start"], b["lens"], D ** -0.5, 0,
                                           b["err"])
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out, ref, mag)
    b = _batch([47, 52], [1, 1], nq, nkv, D, bs, seed=22, shared=32)
    out = torch.ops.spark_b200.attn_shared_prefix(b["q"], b["kc"], b["vc"], b["table"], b["lens"],
                                                  torch.tensor([32], dtype=torch.int32, device="cuda"), D ** -0.5,
                                                  b["err"])
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out, ref, mag)
    qkv = torch.randn((3, (nq + 2 * nkv) * D), device="cuda").to(torch.bfloat16)
    cs = torch.cat([torch.ones((8, 64)), torch.zeros((8, 64))], 1).to(torch.bfloat16).cuda()
    kc, vc = torch.zeros((1, nkv, bs, D), dtype=torch.bfloat16, device="cuda"), torch.zeros(
        (1, nkv, bs, D), dtype=torch.bfloat16, device="cuda")
    at = torch.arange(3, device="cuda")
    q = torch.ops.spark_b200.qk_norm_rope_store_rows(qkv, nq, nkv, D, None, None, 1e-6, cs, at, at, kc, vc, b["err"])
    rows = qkv.view(3, -1, D)
    assert torch.equal(q, rows[:, :nq]) and torch.equal(kc[0, :, :3].transpose(0, 1), rows[:, nq:nq + nkv])
    assert torch.equal(vc[0, :, :3].transpose(0, 1), rows[:, nq + nkv:]) and int(b["err"]) == 0


def test_paged_refusals(cuda):
    import torch
    from spark_b200 import ops
    from spark_b200._lib import SparkError
    nq, nkv, D, bs = 8, 2, 128, 16
    b = _batch([0], [20], nq, nkv, D, bs, seed=30)
    plan = ops.AttnPlan(20, 1, nq, nkv, D)
    out = torch.zeros_like(b["q"])
    args = lambda **k: {**dict(q=b["q"], k_cache=b["kc"], v_cache=b["vc"], block_table=b["table"], plan=plan,  # noqa: E731
                               scale=D ** -0.5, out=out, error=b["err"]), **k}
    with pytest.raises(ValueError):  # no plan made yet
        ops.attn_prompt_out(**args())
    plan.update(b["start"], b["lens"])
    with pytest.raises(ValueError):  # another kind of plan
        ops.attn_shared_prefix_out(**args())
    for bad in (dict(q=b["q"].float()), dict(q=b["q"].cpu()), dict(out=out[:10]), dict(q=b["q"][:, :4]),
                dict(k_cache=b["kc"][:, :, :8]), dict(block_table=b["table"].long()), dict(error=b["err"].long()),
                dict(q=torch.cat([b["q"], b["q"]]), out=torch.cat([out, out])),
                dict(block_table=b["table"][:0])):
        with pytest.raises(ValueError):
            ops.attn_prompt_out(**args(**bad))
    odd = torch.zeros((20, nq, D + 4), dtype=torch.bfloat16, device="cuda")
    for bad in (dict(scale=0.0), dict(scale=float("nan")), dict(q=odd[..., :D]), dict(out=odd[..., :D])):
        with pytest.raises(SparkError):
            ops.attn_prompt_out(**args(**bad))
    small = {"k_cache": torch.zeros((4, nkv, 8, D), dtype=torch.bfloat16, device="cuda")}
    small["v_cache"] = small["k_cache"]
    with pytest.raises(SparkError):  # pages of 8 tokens
        ops.attn_prompt_out(**args(**small))
    for shape in ((20, 1, 8, 3, D), (20, 1, 8, 2, 64), (0, 1, 8, 2, D), (20, 1, 258, 2, D)):
        with pytest.raises(ValueError):
            ops.AttnPlan(*shape)
    with pytest.raises(ValueError):  # more requests than the plan is for
        plan.update(torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        ops.AttnPlan(20, 1, nq, nkv, D, window=5).update_prefix(b["lens"], b["lens"])


@pytest.mark.parametrize("D,nq,nkv", [(128, 8, 2), (256, 8, 2)])
@pytest.mark.parametrize("ctx,new", [([0], [700]), ([2000, 900], [1, 3])])
def test_attn_prompt_large_and_climbing_scores(cuda, D, nq, nkv, ctx, new):
    """Scores up to 10^4 that climb along the keys, so that the softmax's reference moves at
    every tile and by more than any single exponential could take.  q and k are small
    integers: every score is exact in fp32 and the tolerance stays the rounding of p."""
    import torch
    from spark_b200 import ops
    b = _batch(ctx, new, nq, nkv, D, 16, seed=31)
    g = torch.Generator(device="cuda").manual_seed(32)
    b["q"].copy_(torch.randint(0, 2, b["q"].shape, generator=g, device="cuda") * 512)
    for r, m in enumerate(b["len"]):
        at = torch.arange(m, device="cuda")
        blk, off = b["table"][r, at // 16].long(), at % 16
        k = torch.randint(-1, 2, (m, nkv, D), generator=g, device="cuda").float()
        k[:, :, 0] = (at.float() / m * 200).round()[:, None]  # the climb
        b["kc"][blk, :, off] = k.to(torch.bfloat16)
    b["q"][:, :, 0] = 512
    plan = ops.AttnPlan(b["q"].shape[0], len(ctx), nq, nkv, D).update(b["start"], b["lens"])
    out = torch.full_like(b["q"], float("nan"))
    ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    assert int(b["err"]) == 0
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out, ref, mag)


def test_attn_prompt_pages_past_32_bit_offsets(cuda):
    """Caches of more than 2^31 elements, the requests' pages at their far end."""
    import torch
    from spark_b200 import ops
    nq, nkv, D, bs, n = 32, 8, 128, 128, 300
    blocks = 17000  # x 2^17 elements a page
    kc = torch.empty((blocks, nkv, bs, D), dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    assert kc.numel() > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(33)
    ids = [blocks - 1, blocks - 5, blocks - 3, 2, blocks - 2, blocks - 4]
    kc[ids], vc[ids] = (torch.randn((6, nkv, bs, D), generator=g, device="cuda").to(torch.bfloat16) for _ in "kv")
    table = torch.tensor([ids[:3], ids[3:]], dtype=torch.int32, device="cuda")
    i32 = {"dtype": torch.int32, "device": "cuda"}
    start, lens = torch.tensor([0, n, n + 1], **i32), torch.tensor([n, 290], **i32)
    qkv = torch.randn((n + 1, (nq + 2 * nkv) * D), generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.cat([torch.arange(n, device="cuda"), torch.tensor([289], device="cuda")])
    slots = torch.cat([table[0].long()[pos[:n] // bs] * bs + pos[:n] % bs, table[1].long()[2:3] * bs + 289 - 2 * bs])
    cs = torch.cat([torch.ones((400, 64)), torch.zeros((400, 64))], 1).to(torch.bfloat16).cuda()
    q, err = torch.empty((n + 1, nq, D), dtype=torch.bfloat16, device="cuda"), torch.zeros(1, **i32)
    ops.qk_norm_rope_store_rows(qkv, nq, nkv, D, None, None, 0.0, cs, pos, slots, kc, vc, q, err)
    out = torch.zeros_like(q)
    plan = ops.AttnPlan(n + 1, 2, nq, nkv, D).update(start, lens)
    ops.attn_prompt_out(q, kc, vc, table, plan, D ** -0.5, out, err)
    torch.cuda.synchronize()
    assert int(err) == 0
    b = {"q": q, "kc": kc, "vc": vc, "table": table, "new": [n, 1], "len": [n, 290], "bs": bs}
    assert torch.equal(kc[ids[0], :, 5], qkv[5].view(-1, D)[nq:nq + nkv])
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out, ref, mag)


@pytest.mark.parametrize("D,nq,nkv", [(128, 32, 8), (128, 24, 4), (256, 16, 4), (256, 24, 4)])
def test_attn_prompt_same_bits_every_time(cuda, D, nq, nkv):
    """Items of all kinds behind one another in a CTA (rows without tokens, whose warps skip
    what the others wait for; references that move at every tile; parts): 200 replays, one
    result."""
    import torch
    from spark_b200 import ops
    ctx = [0, 2000, 77, 0, 5000, 31] * 12
    new = [1, 3, 200, 130, 1, 33] * 12
    b = _batch(ctx, new, nq, nkv, D, 16, seed=34)
    at = torch.arange(16, device="cuda") / 4  # the reference moves inside a page and from page to page
    b["kc"][:, :, :, 0] = (torch.rand((b["kc"].shape[0], 1, 1), device="cuda") * 60 + at).to(torch.bfloat16).expand(
        b["kc"].shape[:3])
    b["q"][:, :, 0] = 16
    plan = ops.AttnPlan(b["q"].shape[0], len(ctx), nq, nkv, D).update(b["start"], b["lens"])
    out = torch.zeros_like(b["q"])
    ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out, ref, mag)
    want = out.clone()
    differ = torch.zeros(1, dtype=torch.int64, device="cuda")
    for _ in range(200):
        out.zero_()
        ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
        differ += (out.view(torch.int16) != want.view(torch.int16)).sum()
    assert int(differ) == 0 and int(b["err"]) == 0


def test_attn_two_calls_at_once_with_a_plan_each(cuda):
    """Two streams, two captured graphs, replayed together: equal to one after the other."""
    import torch
    from spark_b200 import ops
    nq, nkv, D, bs = 32, 8, 128, 16
    jobs = []
    for seed, (ctx, new) in enumerate([([4000, 100], [1, 1]), ([0, 64], [300, 70])]):
        b = _batch(ctx, new, nq, nkv, D, bs, seed=40 + seed)
        plan = ops.AttnPlan(b["q"].shape[0], 2, nq, nkv, D)
        out = torch.zeros_like(b["q"])

        def step(b=b, plan=plan, out=out):
            plan.update(b["start"], b["lens"])
            ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        # the graph holds the plan's addresses, not the plan: it is kept as long as the graph
        jobs.append((b, out, out.clone(), graph, torch.cuda.Stream(), plan))
    for _ in range(20):
        for b, out, want, graph, stream, _plan in jobs:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                out.zero_()
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for b, out, want, graph, stream, _plan in jobs:
            assert torch.equal(out.view(torch.int16), want.view(torch.int16)) and int(b["err"]) == 0


@pytest.mark.parametrize("D,nq,nkv", [(128, 32, 8), (256, 16, 4)])
def test_attn_wait_that_runs_out_reports_and_recovers(cuda, D, nq, nkv):
    """A wait limit of 0 makes the first unfinished wait give up: the kernel returns, the
    caller's word says so (not 2: copies and products drained, tensor memory was freed), and
    the next call is right."""
    import torch
    from spark_b200 import ops
    b = _batch([3000, 0], [200, 600], nq, nkv, D, 128, seed=50)
    plan = ops.AttnPlan(800, 2, nq, nkv, D).update(b["start"], b["lens"])
    out = torch.zeros_like(b["q"])
    ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"], wait_ns=0)
    torch.cuda.synchronize()
    assert int(b["err"]) == ops.ERR_WAIT
    b["err"].zero_()
    ops.attn_prompt_out(b["q"], b["kc"], b["vc"], b["table"], plan, D ** -0.5, out, b["err"])
    torch.cuda.synchronize()
    assert int(b["err"]) == 0
    ref, mag = _attn_ref(b, nq, nkv, D, D ** -0.5)
    _close(out, ref, mag)


def test_paged_plan_in_a_graph_takes_pages_each_replay(cuda):
    """free_head advanced in place, replay by replay."""
    import torch
    from spark_b200 import ops
    i32 = {"dtype": torch.int32, "device": "cuda"}
    R, bs = 3, 16
    ctx, new = torch.zeros(R, **i32), torch.tensor([16, 5, 0], **i32)
    table, free = torch.full((R, 4), -1, **i32), torch.arange(100, 140, **i32)
    head, counter, err = torch.zeros(1, **i32), torch.zeros(1, **i32), torch.zeros(1, **i32)
    start, lens = torch.zeros(R + 1, **i32), torch.zeros(R, **i32)
    pos, slots = torch.zeros(21, dtype=torch.int64, device="cuda"), torch.zeros(21, dtype=torch.int64, device="cuda")

    def step():
        ops.paged_plan_out(ctx, new, table, bs, start, lens, pos, slots, counter, err, free_blocks=free,
                           free_head=head)
        ctx.copy_(lens)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    # 16 + 5 tokens, four times: 4 pages, and pages at 0, (5 10 15) none, 16 .. 20
    assert int(err) == 0 and ctx.tolist() == [64, 20, 0] and int(head) == 6 and int(counter) == 0
    assert table.tolist() == [[100, 102, 103, 104], [101, 105, -1, -1], [-1] * 4]
    assert pos[16:].tolist() == [15, 16, 17, 18, 19] and slots[16:].tolist() == [101 * 16 + 15] + [
        105 * 16 + i for i in range(4)]
