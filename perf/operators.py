"""Paged-batch operators: the cases they are measured on, their inputs, their plain torch
forms and their results in 64 bits.

Four operators of a serving batch over the paged bf16 KV cache (pages
[blocks, kv heads, block size, head dim]):

  plan    block tables, positions and slot maps from request lengths
  rope    per-head RMS norm of q and k, position rotation and the paged K / V store
  prompt  causal attention of packed sequences over the cache (whole prompts, chunks on
          top of cached context, single tokens), optional sliding window
  prefix  one decode token per request, a long common prefix read once for the batch

Head layouts are those of the two models in spark_b200.config: 32 query / 8 kv heads of
128, and 16 / 4 heads of 256 with a 513-position window and 64 rotated dims.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

BF16 = torch.bfloat16
EPS = 1e-6


def _package():
    pkg = str(Path(__file__).resolve().parents[1] / "spark-vllm-ascend_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from spark_b200 import ops
    return ops


# ------------------------------------------------------------------------------ cases
def listed() -> list[dict]:
    h128 = {"nq": 32, "nkv": 8, "D": 128}
    h256 = {"nq": 16, "nkv": 4, "D": 256}
    return [
        # a decode step of a batch: one token per request, few of them start a page
        {"name": "plan_decode_64", "kind": "plan", "reqs": 64, "ctx": 6144, "new": 1, "bs": 128, "mix": 1},
        # prompts of very different lengths admitted at once, with padding rows behind them
        {"name": "plan_prompts_256", "kind": "plan", "reqs": 256, "ctx": 0, "new": 511, "bs": 128, "mix": 2},
        # the decode step's single row
        {"name": "rope_1", "kind": "rope", "tokens": 1, "norm": False, "rot": 128, "bs": 128, **h128},
        # the standard prompt
        {"name": "rope_2048_norm", "kind": "rope", "tokens": 2048, "norm": True, "rot": 128, "bs": 128, **h128},
        # a packed batch of prompts, the wide heads with a quarter of them rotated
        {"name": "rope_16111_wide", "kind": "rope", "tokens": 16111, "norm": True, "rot": 64, "bs": 128, **h256},
        # the standard prompt, whole
        {"name": "prompt_2048", "kind": "prompt", "reqs": 1, "new": 2048, "ctx": 0, "window": 0, "bs": 128, "mix": 0,
         **h128},
        # prompts of different lengths packed in one call
        {"name": "prompt_packed_8", "kind": "prompt", "reqs": 8, "new": 3001, "ctx": 0, "window": 0, "bs": 128,
         "mix": 3, **h128},
        # a chunk of a long prompt on top of its cached context
        {"name": "prompt_chunk_32k", "kind": "prompt", "reqs": 1, "new": 509, "ctx": 32259, "window": 0, "bs": 128,
         "mix": 0, **h128},
        # the sliding layers of the wide model
        {"name": "prompt_window_wide", "kind": "prompt", "reqs": 3, "new": 2049, "ctx": 700, "window": 513, "bs": 128,
         "mix": 4, **h256},
        # single tokens of a decode batch over long contexts of different lengths
        {"name": "prompt_single_8", "kind": "prompt", "reqs": 8, "new": 1, "ctx": 32767, "window": 0, "bs": 128,
         "mix": 5, **h128},
        # a few requests behind one system prompt
        {"name": "prefix_8_2048", "kind": "prefix", "reqs": 8, "prefix": 2048, "tail": 200, "bs": 128, "mix": 6,
         **h128},
        # many requests behind one long document
        {"name": "prefix_64_32k", "kind": "prefix", "reqs": 64, "prefix": 32768, "tail": 1000, "bs": 128, "mix": 7,
         **h128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["plan", "rope", "prompt", "prompt", "prefix"])
    bs = rng.choice([16, 64, 128, 128])
    heads = rng.choice([(32, 8, 128), (16, 4, 256), (24, 8, 128), (8, 8, 128), (28, 4, 128), (12, 2, 256)])
    nq, nkv, D = heads
    mix = rng.randrange(1, 1 << 20)
    if kind == "plan":
        if rng.random() < 0.5:
            return {"kind": kind, "reqs": _log(rng, 1, 512), "ctx": _log(rng, 16, 32000), "new": 1, "bs": bs,
                    "mix": mix}
        reqs = _log(rng, 1, 256)
        return {"kind": kind, "reqs": reqs, "ctx": rng.choice([0, 0, 1000]), "new": _log(rng, 2, 130000 // reqs),
                "bs": bs, "mix": mix}
    if kind == "rope":
        return {"kind": kind, "tokens": _log(rng, 1, 16000), "norm": rng.random() < 0.6,
                "rot": rng.choice([D, D, D // 2, 64]), "bs": bs, "nq": nq, "nkv": nkv, "D": D}
    if kind == "prompt":
        window = rng.choice([0, 0, 0, 513, 100])
        shape = rng.choice(["whole", "packed", "chunk", "single"])
        if shape == "whole":
            c = {"reqs": 1, "new": _log(rng, 1, 4000), "ctx": 0}
        elif shape == "packed":
            c = {"reqs": rng.randint(2, 12), "new": _log(rng, 16, 2000), "ctx": rng.choice([0, 0, 300])}
        elif shape == "chunk":
            c = {"reqs": rng.randint(1, 2), "new": _log(rng, 8, 256), "ctx": _log(rng, 500, 30000)}
        else:
            c = {"reqs": _log(rng, 1, 32), "new": 1, "ctx": _log(rng, 16, 8000)}
        return {"kind": kind, **c, "window": window, "bs": bs, "mix": mix, "nq": nq, "nkv": nkv, "D": D}
    return {"kind": kind, "reqs": _log(rng, 2, 64), "prefix": _log(rng, 128, 16000) // bs * bs + bs,
            "tail": _log(rng, 2, 800), "bs": bs, "mix": mix, "nq": nq, "nkv": nkv, "D": D}


def _lens(case) -> tuple[list[int], list[int]]:
    """(cached, new) tokens of each request: one request as stated; of several the first as
    stated, the others spread below it."""
    r, mix = case["reqs"], case["mix"]
    rng = random.Random(1000003 * mix + r)
    if case["kind"] == "prefix":
        tails = [case["tail"]] + [rng.randint(1, case["tail"]) for _ in range(r - 1)]
        return [case["prefix"] + t - 1 for t in tails], [1] * r
    new = [case["new"]] + [max(1, int(case["new"] * rng.random() ** 1.5)) for _ in range(r - 1)]
    ctx = [case["ctx"]] + [int(case["ctx"] * rng.uniform(0.3, 1.0)) for _ in range(r - 1)]
    return ctx, new


def _pairs(case) -> int:
    """(query, key) pairs the masks leave, over all requests."""
    total = 0
    for c, n in zip(*_lens(case)):
        w = case.get("window", 0)
        if w:
            total += sum(min(c + i + 1, w) for i in range(n))
        else:
            total += n * c + n * (n + 1) // 2
    return total


def work(case) -> dict:
    kind = case["kind"]
    if kind == "plan":
        ctx, new = _lens(case)
        bs = case["bs"]
        pages = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
        t = sum(new)
        # lengths in; starts, lengths, positions and slots out; a free id read and a table entry written per page
        return {"bytes": 8 * len(new) + 8 * len(new) + 4 + 16 * t + 8 * pages, "flops": 0}
    nq, nkv, D = case["nq"], case["nkv"], case["D"]
    if kind == "rope":
        t = case["tokens"]
        row = (nq + 2 * nkv) * D * 2
        return {"bytes": t * (2 * row + 16 + case["rot"] * 2), "flops": t * (nq + nkv) * D * 8}
    ctx, new = _lens(case)
    t = sum(new)
    qo = 2 * t * nq * D * 2
    if kind == "prompt":
        w = case["window"]
        keys = sum(min(c + n, w + n - 1) if w else c + n for c, n in zip(ctx, new))
        return {"bytes": qo + keys * nkv * D * 4, "flops": 4 * D * nq * _pairs(case)}
    keys = case["prefix"] + sum(c + 1 - case["prefix"] for c in ctx)
    return {"bytes": qo + keys * nkv * D * 4, "flops": 4 * D * nq * sum(c + 1 for c in ctx)}


# ------------------------------------------------------------------------------ inputs
def _pages(n: int, bs: int) -> int:
    return -(-n // bs)


def _tables(case, gen) -> tuple[torch.Tensor, int]:
    """Block tables over a shuffled pool with some spare pages; of a shared prefix every
    request's table begins with the same pages."""
    ctx, new = _lens(case)
    bs = case["bs"]
    need = [_pages(c + n, bs) for c, n in zip(ctx, new)]
    shared = case["prefix"] // bs if case["kind"] == "prefix" else 0
    blocks = shared + sum(n - shared for n in need) + 5
    perm = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device="cuda")
    off = shared
    for r, n in enumerate(need):
        table[r, :shared] = perm[:shared]
        table[r, shared:n] = perm[off:off + n - shared]
        off += n - shared
    return table, blocks


def _normal(shape, gen) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(BF16)


def _inputs(case, seed) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, bs = case["kind"], case["bs"]
    i32 = {"dtype": torch.int32, "device": "cuda"}
    if kind == "plan":
        ctx, new = _lens(case)
        need = [_pages(c + n, bs) for c, n in zip(ctx, new)]
        have = [_pages(c, bs) for c in ctx]
        blocks = sum(need) + 100
        perm = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((len(need), max(need) + 2), -1, **i32)
        off = 0
        for r, n in enumerate(have):
            table[r, :n] = perm[off:off + n]
            off += n
        # the free list: a few ids in front are taken already
        head = 7
        free = torch.cat([torch.full((head,), -1, **i32), perm[off:]])
        return {"ctx": torch.tensor(ctx, **i32), "new": torch.tensor(new, **i32), "table": table, "free": free,
                "head": torch.tensor([head], **i32), "rows": _pages(sum(new), 64) * 64}
    nq, nkv, D = case["nq"], case["nkv"], case["D"]
    if kind == "rope":
        t, rot = case["tokens"], case["rot"]
        blocks = _pages(t, bs) + 3
        max_pos = max(40960, t)
        inv = 1.0 / (1.0e6 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot))
        ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv[None]
        cos_sin = torch.cat([ang.cos(), ang.sin()], -1).to(BF16).cuda()
        first = int(torch.randint(0, max_pos - t + 1, (1,), generator=gen, device="cuda"))
        slots = torch.randperm(blocks * bs, generator=gen, device="cuda")[:t].contiguous()
        gamma = (lambda: (1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).to(BF16)) if case["norm"] else \
            (lambda: None)
        return {"qkv": _normal((t, (nq + 2 * nkv) * D), gen), "qg": gamma(), "kg": gamma(), "cos_sin": cos_sin,
                "pos": torch.arange(first, first + t, device="cuda"), "slots": slots,
                "k_cache": _normal((blocks, nkv, bs, D), gen), "v_cache": _normal((blocks, nkv, bs, D), gen)}
    ctx, new = _lens(case)
    table, blocks = _tables(case, gen)
    t = sum(new)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return {"q": _normal((t, nq, D), gen), "k_cache": _normal((blocks, nkv, bs, D), gen),
            "v_cache": _normal((blocks, nkv, bs, D), gen), "table": table, "start": torch.tensor(start, **i32),
            "lens": torch.tensor([c + n for c, n in zip(ctx, new)], **i32),
            "prefix": torch.tensor([case.get("prefix", 0)], **i32)}


def prepare(case, seed) -> dict:
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if kind == "plan":
        r, t = case["reqs"], s["rows"]
        s["out"] = {"query_start": torch.zeros(r + 1, dtype=torch.int32, device="cuda"),
                    "seq_lens": torch.zeros(r, dtype=torch.int32, device="cuda"),
                    "positions": torch.zeros(t, dtype=torch.int64, device="cuda"),
                    "slot_mapping": torch.zeros(t, dtype=torch.int64, device="cuda"),
                    "free_head": torch.zeros(1, dtype=torch.int32, device="cuda")}
    elif kind == "rope":
        s["q"] = torch.zeros((case["tokens"], case["nq"], case["D"]), dtype=BF16, device="cuda")
    else:
        s["o"] = torch.zeros_like(s["q"])
        s["lists"] = _lens(case)
    if own:
        ops = _package()
        s["ops"] = ops
        s["error"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        if kind == "plan":
            s["counter"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        elif kind in ("prompt", "prefix"):  # one plan per step serves every layer
            plan = ops.AttnPlan(s["q"].shape[0], case["reqs"], case["nq"], case["nkv"], case["D"], device="cuda",
                                window=case.get("window", 0))
            if kind == "prompt":
                plan.update(s["start"], s["lens"])
            else:
                plan.update_prefix(s["lens"], s["prefix"])
            s["plan"] = plan
    return s


# ------------------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"plan": _own_plan, "rope": _own_rope, "prompt": _own_prompt, "prefix": _own_prefix}[kind](state)
    return {"plan": _plain_plan, "rope": _plain_rope, "prompt": _plain_attention, "prefix": _plain_attention}[kind](
        state)


def _own_plan(s):
    o = s["out"]
    s["ops"].paged_plan_out(s["ctx"], s["new"], s["table"], s["case"]["bs"], o["query_start"], o["seq_lens"],
                            o["positions"], o["slot_mapping"], s["counter"], s["error"], free_blocks=s["free"],
                            free_head=s["head"], free_head_out=o["free_head"])
    return {**o, "table": s["table"]}


def _own_rope(s):
    c = s["case"]
    s["ops"].qk_norm_rope_store_rows(s["qkv"], c["nq"], c["nkv"], c["D"], s["qg"], s["kg"], EPS, s["cos_sin"],
                                     s["pos"], s["slots"], s["k_cache"], s["v_cache"], s["q"], s["error"])
    return {"q": s["q"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_prompt(s):
    return s["ops"].attn_prompt_out(s["q"], s["k_cache"], s["v_cache"], s["table"], s["plan"],
                                    s["case"]["D"] ** -0.5, s["o"], s["error"])


def _own_prefix(s):
    return s["ops"].attn_shared_prefix_out(s["q"], s["k_cache"], s["v_cache"], s["table"], s["plan"],
                                           s["case"]["D"] ** -0.5, s["o"], s["error"])


def _plain_plan(s):
    bs, ctx, new = s["case"]["bs"], s["ctx"].long(), s["new"].long()
    table, t = s["table"], s["rows"]
    lens = ctx + new
    end = torch.cumsum(new, 0)
    start = end - new
    have, need = (ctx + bs - 1) // bs, (lens + bs - 1) // bs
    taken = torch.cumsum(need - have, 0)
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    src = s["head"].long() + (taken - (need - have))[:, None] + col - have[:, None]
    ids = s["free"][src.clamp(0, s["free"].numel() - 1)]
    table.copy_(torch.where(fresh, ids, table))
    row = torch.arange(t, device=table.device)
    req = torch.searchsorted(end, row, right=True)
    live = req < ctx.numel()
    req = req.clamp(max=ctx.numel() - 1)
    pos = torch.where(live, ctx[req] + row - start[req], 0)
    slot = torch.where(live, table[req, pos // bs].long() * bs + pos % bs, -1)
    o = s["out"]
    o["query_start"][0] = 0
    o["query_start"][1:] = end.int()
    o["seq_lens"].copy_(lens.int())
    o["positions"].copy_(pos)
    o["slot_mapping"].copy_(slot)
    o["free_head"].copy_((s["head"].long() + taken[-1:]).int())
    return {**o, "table": table}


def _plain_rope(s):
    c = s["case"]
    nq, nkv, D, rot, bs, t = c["nq"], c["nkv"], c["D"], c["rot"], c["bs"], c["tokens"]
    x = s["qkv"].float().view(t, nq + 2 * nkv, D)
    qk, v = x[:, :nq + nkv], x[:, nq + nkv:]
    if c["norm"]:
        g = torch.cat([s["qg"].float().expand(nq, D), s["kg"].float().expand(nkv, D)])
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * g
    half = rot // 2
    cs = s["cos_sin"][s["pos"]].float()[:, None, :]
    cos, sin = cs[..., :half], cs[..., half:]
    a, b = qk[..., :half], qk[..., half:rot]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin, qk[..., rot:]], -1)
    s["q"].copy_(qk[:, :nq])
    blk, off = s["slots"] // bs, s["slots"] % bs
    s["k_cache"][blk, :, off] = qk[:, nq:].to(BF16)
    s["v_cache"][blk, :, off] = v.to(BF16)
    return {"q": s["q"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    """Scores, softmax and the weighted sum of each request in 32 bits, a kv head at a time."""
    c = s["case"]
    nq, nkv, D, bs, window = c["nq"], c["nkv"], c["D"], c["bs"], c.get("window", 0)
    g, scale = nq // nkv, c["D"] ** -0.5
    t0 = 0
    for r, (cached, n) in enumerate(zip(*s["lists"])):
        m = cached + n
        lo = max(0, cached + 1 - window) if window else 0
        pages = s["table"][r, lo // bs:_pages(m, bs)].long()
        base = lo // bs * bs
        kpos = torch.arange(base, m, device="cuda")
        qpos = torch.arange(cached, m, device="cuda")
        keep = kpos[None, :] <= qpos[:, None]
        if window:
            keep = keep & (kpos[None, :] > qpos[:, None] - window)
        q = s["q"][t0:t0 + n].float().view(n, nkv, g, D)
        for h in range(nkv):
            k = s["k_cache"][pages, h].float().view(-1, D)[:m - base]
            v = s["v_cache"][pages, h].float().view(-1, D)[:m - base]
            p = (q[:, h].reshape(n * g, D) @ k.t()).view(n, g, -1) * scale
            p = p.masked_fill(~keep[:, None, :], float("-inf"))
            p = torch.exp(p - p.amax(-1, keepdim=True))
            o = (p.view(n * g, -1) @ v) / p.sum(-1).view(n * g, 1)
            s["o"][t0:t0 + n, h * g:(h + 1) * g] = o.view(n, g, D).to(BF16)
        t0 += n
    return s["o"]


# ------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    kind, bs = case["kind"], case["bs"]
    if kind == "plan":
        ctx, new = _lens(case)
        free, head, table = s["free"].tolist(), int(s["head"]), s["table"].tolist()
        start, pos, slot = [0], [], []
        for r, (c, n) in enumerate(zip(ctx, new)):
            for p in range(_pages(c, bs), _pages(c + n, bs)):
                table[r][p] = free[head]
                head += 1
            for x in range(c, c + n):
                pos.append(x)
                slot.append(table[r][x // bs] * bs + x % bs)
            start.append(start[-1] + n)
        pad = s["rows"] - len(pos)
        i32 = {"dtype": torch.int32, "device": "cuda"}
        return {"query_start": torch.tensor(start, **i32),
                "seq_lens": torch.tensor([c + n for c, n in zip(ctx, new)], **i32),
                "positions": torch.tensor(pos + [0] * pad, device="cuda"),
                "slot_mapping": torch.tensor(slot + [-1] * pad, device="cuda"),
                "free_head": torch.tensor([head], **i32), "table": torch.tensor(table, **i32)}
    nq, nkv, D = case["nq"], case["nkv"], case["D"]
    if kind == "rope":
        t, half = case["tokens"], case["rot"] // 2
        heads = s["qkv"].double().unflatten(1, (nq + 2 * nkv, D))
        cs = s["cos_sin"].double()[s["pos"]]
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        q = torch.empty((t, nq, D), dtype=torch.float64, device="cuda")
        blk, off = torch.div(s["slots"], bs, rounding_mode="floor"), s["slots"].remainder(bs)
        for h in range(nq + nkv):
            x = heads[:, h]
            gamma = s["qg"] if h < nq else s["kg"]
            if gamma is not None:
                x = gamma.double() * x / (x.square().sum(1, keepdim=True) / D + EPS).sqrt()
            y = x.clone()
            y[:, :half] = x[:, :half] * cs[:, :half] - x[:, half:2 * half] * cs[:, half:]
            y[:, half:2 * half] = x[:, half:2 * half] * cs[:, :half] + x[:, :half] * cs[:, half:]
            if h < nq:
                q[:, h] = y
            else:
                kc[blk, h - nq, off] = y
        for h in range(nkv):
            vc[blk, h, off] = heads[:, nq + nkv + h]
        return {"q": q, "k_cache": kc, "v_cache": vc}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    start, lens = s["start"].tolist(), s["lens"].tolist()
    window = case.get("window", 0) or 1 << 30
    for r, m in enumerate(lens):
        i0, i1 = start[r], start[r + 1]
        where = torch.arange(m, device="cuda")
        blk, off = s["table"][r].long()[where // bs], where % bs
        for h in range(nq):
            k, v = s["k_cache"][blk, h * nkv // nq, off].double(), s["v_cache"][blk, h * nkv // nq, off].double()
            for a in range(i0, i1, 1024):  # query rows a .. b at positions m - (i1 - a) ..
                b = min(i1, a + 1024)
                at = m - i1 + torch.arange(a, b, device="cuda")
                x = s["q"][a:b, h].double() @ k.t() / math.sqrt(D)
                behind = at[:, None] - where[None, :]
                x[(behind < 0) | (behind >= window)] = float("-inf")
                out[a:b, h] = torch.softmax(x, 1) @ v
    return out
