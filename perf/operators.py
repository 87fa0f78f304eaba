"""Workloads of the paged K/V cache operators: page bookkeeping, the cache write and the attention that reads it.

``listed()`` gives the cases, ``draw(rng)`` more of the same ranges, ``prepare`` a case's inputs on the GPU, ``run``
one pass (the operators of ``hspmn_b200.ops`` when ``own`` is true, otherwise their plain form in elementary torch
operations), ``work`` what a pass cannot do without, and ``exact`` the same outputs from the definitions in 64 bits.
"""

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def listed():
    heads = {"H": 16, "Hkv": 4, "hd": 128}  # the block's benchmark configuration (dim 2048)
    return [
        # one decode step of 64 requests: pages and slots for one new token each
        {"name": "slots_decode_64", "op": "slots", "requests": 64, "ctx_lo": 1, "ctx_hi": 32768, "new_lo": 1, "new_hi": 1,
         "single": 1.0, "page": 64, "pad": 0, "mix": 11},
        # many ragged prompts admitted at once, token count padded as for a captured step
        {"name": "slots_prompts_509", "op": "slots", "requests": 509, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 1,
         "new_hi": 4096, "single": 0.0, "page": 16, "pad": 301, "mix": 12},
        # the decode step's cache write
        {"name": "write_decode_61", "op": "write", "requests": 61, "ctx_lo": 1, "ctx_hi": 2048, "new_lo": 1, "new_hi": 1,
         "single": 1.0, "page": 64, "joint": False, "tables": "same", "dtype": "bf16", "mix": 21, **heads},
        # prompt chunks of 16 sequences of up to the benchmark's length
        {"name": "write_prompts_bf16", "op": "write", "requests": 16, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 4096,
         "new_hi": 4096, "single": 0.0, "page": 64, "joint": False, "tables": "same", "dtype": "bf16", "mix": 22, **heads},
        # ragged chunks of the default configuration (dim 768), float32 tables, K and V in one allocation
        {"name": "write_ragged_f16", "op": "write", "requests": 33, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 17,
         "new_hi": 2048, "single": 0.0, "page": 16, "joint": True, "tables": "f32", "dtype": "f16", "mix": 23,
         "H": 12, "Hkv": 4, "hd": 64},
        # one user, one token, a short answer: the smallest call
        {"name": "attend_one_token_500", "op": "attend", "requests": 1, "ctx_lo": 500, "ctx_hi": 500, "new_lo": 1,
         "new_hi": 1, "single": 1.0, "routed": 1.0, "page": 16, "joint": False, "dtype": "bf16", "mix": 31, "H": 12,
         "Hkv": 4, "hd": 64},
        # a full decode batch with ragged contexts
        {"name": "attend_decode_64", "op": "attend", "requests": 64, "ctx_lo": 1024, "ctx_hi": 32768, "new_lo": 1,
         "new_hi": 1, "single": 1.0, "routed": 1.0, "page": 64, "joint": False, "dtype": "bf16", "mix": 32, **heads},
        # one token over the longest context the framework runs
        {"name": "attend_decode_262144", "op": "attend", "requests": 1, "ctx_lo": 262143, "ctx_hi": 262143, "new_lo": 1,
         "new_hi": 1, "single": 1.0, "routed": 1.0, "page": 128, "joint": False, "dtype": "bf16", "mix": 33, **heads},
        # decode without head grouping, float16, small pages, K and V in one allocation
        {"name": "attend_decode_37_mha_f16", "op": "attend", "requests": 37, "ctx_lo": 129, "ctx_hi": 8192, "new_lo": 1,
         "new_hi": 1, "single": 1.0, "routed": 1.0, "page": 16, "joint": True, "dtype": "f16", "mix": 34, "H": 16,
         "Hkv": 16, "hd": 64},
        # whole prompts, every token a query (packed, ragged lengths, empty cache before)
        {"name": "attend_prompts_dense", "op": "attend", "requests": 7, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 511,
         "new_hi": 4096, "single": 0.0, "routed": 1.0, "page": 64, "joint": False, "dtype": "bf16", "mix": 35, **heads},
        # the router's fifth of a long prompt's chunk over what is cached already: the largest call
        {"name": "attend_chunk_routed", "op": "attend", "requests": 3, "ctx_lo": 24576, "ctx_hi": 24576, "new_lo": 8192,
         "new_hi": 8192, "single": 0.0, "routed": 0.2, "page": 64, "joint": False, "dtype": "bf16", "mix": 36, **heads},
        # decode tokens and prompt chunks in one batch
        {"name": "attend_mixed_52_f16", "op": "attend", "requests": 52, "ctx_lo": 65, "ctx_hi": 8192, "new_lo": 255,
         "new_hi": 1024, "single": 0.9, "routed": 1.0, "page": 32, "joint": True, "dtype": "f16", "mix": 37, **heads},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def _lens(case):
    """(cached, new) tokens of each request; they belong to the case, not to the seed."""
    rng = random.Random(case["mix"])
    ctx, new = [], []
    for _ in range(case["requests"]):
        ctx.append(0 if case["ctx_hi"] == 0 else _log_between(rng, max(1, case["ctx_lo"]), case["ctx_hi"]))
        new.append(1 if rng.random() < case["single"] else _log_between(rng, case["new_lo"], case["new_hi"]))
    return ctx, new


def _queries(case):
    """Query rows of each request: the router's share of its new tokens, one at least."""
    return [max(1, int(n * case["routed"])) for n in _lens(case)[1]]


def work(case):
    ctx, new = _lens(case)
    n, r, p = sum(new), case["requests"], case["page"]
    if case["op"] == "slots":
        fresh = sum(-(-(c + m) // p) - -(-c // p) for c, m in zip(ctx, new))
        # lengths in, offsets and lengths out, a page number in and out for each fresh page, position and slot out
        return {"bytes": 8 * r + 4 * (r + 1) + 4 * r + 8 * fresh + 16 * (n + case["pad"]) + 4, "flops": 0}
    es = 4 if case["dtype"] == "f32" else 2
    row = case["Hkv"] * case["hd"] * es
    if case["op"] == "write":
        tab = case["hd"] * (4 if case["tables"] == "f32" else es)
        # K and V in and out, position and slot in, each table row that is met once
        return {"bytes": 4 * n * row + 16 * n + 2 * tab * min(n, max(c + m for c, m in zip(ctx, new))),
                "flops": 3 * n * case["Hkv"] * case["hd"]}
    q = _queries(case)
    pairs = 0
    for c, m, k in zip(ctx, new, q):
        # the k query positions are spread evenly over the new tokens, the last one among them
        pairs += k * (c + m) - (m / k) * (k * (k - 1) / 2)
    kv = sum(c + m for c, m in zip(ctx, new))
    return {"bytes": 2 * kv * row + 2 * sum(q) * case["H"] * case["hd"] * es + 8 * sum(q) + 4 * (kv // p + 2 * r),
            "flops": int(4 * case["hd"] * case["H"] * pairs)}


_HEADS = ((16, 4, 128), (16, 16, 128), (12, 4, 64), (8, 2, 128), (16, 16, 64), (6, 2, 64), (8, 8, 96), (4, 1, 128))


def draw(rng):
    most = max((work(c) for c in listed() if c["op"] == "attend"), key=lambda w: w["flops"])["flops"]
    while True:
        op = rng.choice(("slots", "write", "attend", "attend", "attend"))
        h, hkv, hd = rng.choice(_HEADS)
        case = {"op": op, "requests": _log_between(rng, 1, 509 if op == "slots" else 64), "page": rng.choice((16, 32, 64, 128)),
                "single": rng.choice((0.0, 1.0, 0.7)), "mix": rng.randrange(1 << 30)}
        case["ctx_hi"] = rng.choice((0, 1, 1, 1)) * _log_between(rng, 64, 32768)
        case["ctx_lo"] = min(case["ctx_hi"], max(1, case["ctx_hi"] // rng.choice((1, 4, 64))))
        case["new_hi"] = _log_between(rng, 2, 4096)
        case["new_lo"] = max(1, case["new_hi"] // rng.choice((1, 4, 64)))
        if op == "slots":
            case["pad"] = rng.choice((0, rng.randrange(1, 512)))
            if sum(_lens(case)[1]) > 600_000:
                continue
            return case
        case.update(H=h, Hkv=hkv, hd=hd, dtype=rng.choice(("bf16", "f16")), joint=rng.random() < 0.5)
        if op == "write":
            case["ctx_hi"], case["ctx_lo"] = min(case["ctx_hi"], 4096), min(case["ctx_lo"], 4096)
            case.update(tables=rng.choice(("same", "f32")))
            if work(case)["bytes"] > 280_000_000:
                continue
            return case
        case["routed"] = rng.choice((1.0, 1.0, 0.2))
        ctx, new = _lens(case)
        longest = max(c + m for c, m in zip(ctx, new))
        if case["requests"] * h * max(_queries(case)) * longest > 2 << 30 or work(case)["flops"] > most:
            continue
        if case["requests"] * longest * hkv * hd > 1 << 30:
            continue
        return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _tables(length, hd, dtype, dev):
    """Rotary cos / sin rows of positions 0 .. length-1 (base 10000), angles in 64 bits."""
    inv = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, dtype=torch.float64, device=dev) / hd))
    ang = torch.outer(torch.arange(length, dtype=torch.float64, device=dev), inv)
    ang = torch.cat((ang, ang), dim=-1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def _cache(case, pages, gen, dev, dtype):
    """K and V caches [pages, page, Hkv, hd]: two allocations, or the halves of one."""
    shape = (case["page"], case["Hkv"], case["hd"])
    if case["joint"]:
        kv = torch.randn((pages, 2) + shape, generator=gen, device=dev, dtype=dtype)
        return kv[:, 0], kv[:, 1]
    return (torch.randn((pages,) + shape, generator=gen, device=dev, dtype=dtype),
            torch.randn((pages,) + shape, generator=gen, device=dev, dtype=dtype))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    ctx, new = _lens(case)
    p, r, n = case["page"], case["requests"], sum(new)
    i32 = {"dtype": torch.int32, "device": dev}
    held = [-(-c // p) for c in ctx]
    total = [-(-(c + m) // p) for c, m in zip(ctx, new)]
    s = {"op": case["op"], "page": p, "n": n, "longest": max(c + m for c, m in zip(ctx, new))}
    if case["op"] == "slots":
        spare = 5
        pages = sum(total) + spare
        order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
        table = torch.full((r, max(total) + 1), -1, **i32)
        col = torch.arange(table.shape[1], device=dev)
        held_t = torch.tensor(held, device=dev)
        first = torch.cumsum(held_t, 0) - held_t
        inside = col[None, :] < held_t[:, None]
        table = torch.where(inside, order[(first[:, None] + col[None, :]).clamp(max=pages - 1)], table)
        s.update(block_table=table, seq_lens=torch.tensor(ctx, **i32), new_lens=torch.tensor(new, **i32),
                 free_pages=order[sum(held):].clone(), tokens=n + case["pad"])
        return s
    dtype = _DTYPES[case["dtype"]]
    pages = sum(total) + 3
    order = torch.randperm(pages, generator=gen, device=dev)
    width = max(total)
    table = torch.full((r, width), -1, **i32)
    col = torch.arange(width, device=dev)
    total_t = torch.tensor(total, device=dev)
    first = torch.cumsum(total_t, 0) - total_t
    inside = col[None, :] < total_t[:, None]
    table = torch.where(inside, order[(first[:, None] + col[None, :]).clamp(max=pages - 1)].to(torch.int32), table)
    s["k_cache"], s["v_cache"] = _cache(case, pages, gen, dev, dtype)
    ctx_t, new_t = torch.tensor(ctx, device=dev), torch.tensor(new, device=dev)
    if case["op"] == "write":
        req = torch.repeat_interleave(torch.arange(r, device=dev), new_t, output_size=n)
        pos = torch.arange(n, device=dev) - (torch.cumsum(new_t, 0) - new_t)[req] + ctx_t[req]
        s["positions"] = pos
        s["slots"] = table[req, pos // p].to(torch.int64) * p + pos % p
        s["k"] = torch.randn((n, case["Hkv"], case["hd"]), generator=gen, device=dev, dtype=dtype)
        s["v"] = torch.randn((n, case["Hkv"], case["hd"]), generator=gen, device=dev, dtype=dtype)
        s["cos"], s["sin"] = _tables(s["longest"], case["hd"], torch.float32 if case["tables"] == "f32" else dtype, dev)
        return s
    q = _queries(case)
    cu = [0]
    for k in q:
        cu.append(cu[-1] + k)
    q_t = torch.tensor(q, device=dev)
    req = torch.repeat_interleave(torch.arange(r, device=dev), q_t, output_size=cu[-1])
    at = torch.arange(cu[-1], device=dev) - (torch.cumsum(q_t, 0) - q_t)[req]
    # the last of k equal parts of the new tokens ends at the last token; distinct and ascending
    s["positions"] = ctx_t[req] + ((at + 1) * new_t[req]) // q_t[req] - 1
    s.update(q=torch.randn((cu[-1], case["H"], case["hd"]), generator=gen, device=dev, dtype=dtype), block_table=table,
             kv_lens=(ctx_t + new_t).to(torch.int32), cu_q=torch.tensor(cu, **i32), max_q=max(q), rows=cu[-1],
             scale=1.0 / math.sqrt(case["hd"]))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


_ops = None


def run(s):
    if own:
        global _ops
        if _ops is None:
            sys.path.insert(0, os.path.join(os.getcwd(), "hspmn-v2.1_b200"))
            from hspmn_b200 import ops as _ops
        ops = _ops
        if s["op"] == "slots":
            cu, kv_lens, positions, slots, taken = ops.paged_slots_(
                s["block_table"], s["seq_lens"], s["new_lens"], s["free_pages"], s["page"], s["tokens"])
            return {"block_table": s["block_table"], "cu": cu, "kv_lens": kv_lens, "positions": positions, "slots": slots,
                    "taken": taken}
        if s["op"] == "write":
            ops.rope_paged_write_(s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_cache"],
                                  s["v_cache"])
            return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return {"o": ops.sqdk_paged_fwd(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_lens"], s["cu_q"],
                                        s["positions"], s["scale"], s["max_q"])}
    return {"slots": _plain_slots, "write": _plain_write, "attend": _plain_attend}[s["op"]](s)


def _plain_slots(s):
    table, seq, new, p = s["block_table"], s["seq_lens"].long(), s["new_lens"].long(), s["page"]
    dev, (r, width), n = table.device, table.shape, s["tokens"]
    ends = torch.cumsum(new, 0)
    cu = torch.cat((ends.new_zeros(1), ends))
    old = (seq + p - 1) // p
    need = (seq + new + p - 1) // p - old
    base = torch.cumsum(need, 0) - need
    col = torch.arange(width, device=dev)[None, :] - old[:, None]
    fresh = (col >= 0) & (col < need[:, None])
    picked = s["free_pages"][(base[:, None] + col).clamp(0, s["free_pages"].shape[0] - 1)]
    table.copy_(torch.where(fresh, picked, table))
    t = torch.arange(n, device=dev)
    req = torch.searchsorted(ends, t, right=True).clamp(max=r - 1)
    inside = t < ends[-1]
    pos = torch.where(inside, seq[req] + t - cu[req], torch.full_like(t, -1))
    page = table[req, pos.clamp(min=0) // p].long()
    slots = torch.where(inside, page * p + pos % p, torch.full_like(t, -1))
    return {"block_table": table, "cu": cu.to(torch.int32), "kv_lens": (seq + new).to(torch.int32), "positions": pos,
            "slots": slots, "taken": need.sum().to(torch.int32).reshape(1)}


def _plain_write(s):
    k, p = s["k"].float(), s["page"]
    cos, sin = s["cos"].float()[s["positions"]][:, None], s["sin"].float()[s["positions"]][:, None]
    half = k.shape[-1] // 2
    turned = torch.cat((-k[..., half:], k[..., :half]), dim=-1)
    page, off = s["slots"] // p, s["slots"] % p
    s["k_cache"][page, off] = (k * cos + turned * sin).to(s["k_cache"].dtype)
    s["v_cache"][page, off] = s["v"]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    q, table, cu, lens = s["q"], s["block_table"].long(), s["cu_q"].long(), s["kv_lens"].long()
    dev, (n, h, hd), (r, _) = q.device, q.shape, table.shape
    hkv, keys, most = s["k_cache"].shape[2], s["longest"], s["max_q"]
    # the requests' keys, values and queries in rows of one length
    pages = table.clamp(min=0)
    k = s["k_cache"][pages].flatten(1, 2)[:, :keys].float().permute(0, 2, 3, 1)
    v = s["v_cache"][pages].flatten(1, 2)[:, :keys].float().transpose(1, 2)
    at = cu[:-1, None] + torch.arange(most, device=dev)[None, :]
    there = at < cu[1:, None]
    at = at.clamp(max=n - 1)
    qs = q[at].float().view(r, most, hkv, h // hkv, hd).permute(0, 2, 3, 1, 4).reshape(r, hkv, -1, hd)
    scores = (qs @ k).view(r, hkv, h // hkv, most, keys).mul_(s["scale"])
    m = torch.arange(keys, device=dev)
    seen = (m[None, None, :] <= s["positions"][at][:, :, None]) & (m[None, None, :] < lens[:, None, None])
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    scores.div_(scores.sum(-1, keepdim=True))
    o = (scores.view(r, hkv, -1, keys) @ v).view(r, hkv, h // hkv, most, hd).permute(0, 3, 1, 2, 4).reshape(r, most, h, hd)
    rows = torch.arange(n, device=dev)
    req = torch.searchsorted(cu[1:], rows, right=True)
    return {"o": o[req, rows - cu[req]].to(q.dtype)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    ctx, new = _lens(case)
    p = case["page"]
    if case["op"] == "slots":
        table, free = s["block_table"].tolist(), s["free_pages"].tolist()
        cu, positions, slots, taken = [0], [], [], 0
        for i, (c, m) in enumerate(zip(ctx, new)):
            for j in range(-(-c // p), -(-(c + m) // p)):
                table[i][j] = free[taken]
                taken += 1
            cu.append(cu[-1] + m)
            positions += range(c, c + m)
            slots += [table[i][t // p] * p + t % p for t in range(c, c + m)]
        pad = [-1] * case["pad"]
        return {"block_table": torch.tensor(table, dtype=torch.int32), "cu": torch.tensor(cu, dtype=torch.int32),
                "kv_lens": torch.tensor([c + m for c, m in zip(ctx, new)], dtype=torch.int32),
                "positions": torch.tensor(positions + pad), "slots": torch.tensor(slots + pad),
                "taken": torch.tensor([taken], dtype=torch.int32)}
    if case["op"] == "write":
        kc, vc = s["k_cache"].double().contiguous(), s["v_cache"].double().contiguous()
        x, half = s["k"].double(), case["hd"] // 2
        cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
        rows = torch.empty_like(x)
        rows[..., :half] = x[..., :half] * cos[:, None, :half] - x[..., half:] * sin[:, None, :half]
        rows[..., half:] = x[..., half:] * cos[:, None, half:] + x[..., :half] * sin[:, None, half:]
        kc.view((-1,) + kc.shape[2:])[s["slots"]] = rows
        vc.view((-1,) + vc.shape[2:])[s["slots"]] = s["v"].double()
        return {"k_cache": kc, "v_cache": vc}
    o = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group, at = case["H"] // case["Hkv"], 0
    for i, (c, m, rows) in enumerate(zip(ctx, new, _queries(case))):
        pages = s["block_table"][i, : -(-(c + m) // p)].long()
        pos = s["positions"][at:at + rows]
        hidden = torch.arange(c + m, device=pos.device)[None, :] > pos[:, None]
        for g in range(case["Hkv"]):
            k = s["k_cache"][pages, :, g].double().reshape(-1, case["hd"])[: c + m]
            v = s["v_cache"][pages, :, g].double().reshape(-1, case["hd"])[: c + m]
            for h in range(g * group, (g + 1) * group):
                w = (s["q"][at:at + rows, h].double() @ k.T) * s["scale"]
                w = torch.softmax(w.masked_fill_(hidden, -math.inf), dim=-1)
                o[at:at + rows, h] = w @ v
        at += rows
    return {"o": o}
