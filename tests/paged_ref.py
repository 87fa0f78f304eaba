"""Plain 64-bit forms of the paged K/V cache operators, for the tests."""

import math

import torch


def slots_ref(table, seq_lens, new_lens, free_pages, page, n):
    """paged_slots_ on lists; ``table`` is a list of rows. Returns the results
    and the new table."""
    table = [list(row) for row in table]
    width = len(table[0]) if table else 0
    cu, kv, positions, slots, taken = [0], [], [], [], 0
    for r, (c, m) in enumerate(zip(seq_lens, new_lens)):
        c, m = max(c, 0), max(m, 0)
        for j in range(min(-(-c // page), width), min(-(-(c + m) // page), width)):
            table[r][j] = free_pages[taken] if taken < len(free_pages) else -1
            taken += 1
        cu.append(cu[-1] + m)
        kv.append(c + m)
        for p in range(c, c + m):
            pg = table[r][p // page] if p // page < width else -1
            positions.append(p)
            slots.append(pg * page + p % page if pg >= 0 else -1)
    positions, slots = positions[:n], slots[:n]
    pad = [-1] * (n - len(positions))
    return table, cu, kv, positions + pad, slots + pad, taken


def rope_ref(k, cos, sin, positions):
    """(rotated K in float64, sum of the two products' sizes)."""
    x, half = k.double(), k.shape[-1] // 2
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    turned = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * c + turned * s, (x * c).abs() + (turned * s).abs()


def weighted(w, v, hidden):
    """sum over the visible keys of w v; a hidden key's infinity or NaN does not count."""
    wild = ~torch.isfinite(v).all(-1)
    if not wild.any():
        return w @ v
    out = w[..., ~wild] @ v[~wild]
    for m in torch.nonzero(wild).flatten().tolist():
        out = out + torch.where(hidden[..., m, None], 0.0, w[..., m, None] * v[m])
    return out


def attend_ref(q, k_cache, v_cache, table, kv_lens, cu_q, positions, scale):
    """sqdk_paged_fwd in float64 and, per output, a bound on the error of a
    kernel that multiplies 16-bit operands, sums in float32 and rounds P and O
    to the operands' type.

    With u half a step of the type, w the softmax weights and e = 2^-23 (one
    float32 operation, rounded or truncated):
      scores    hd products and sums, scale and maximum: (hd + 4) e sum|q k| scale
                in the exponent, so that much of each weight, and as much again in
                the row sum; the exponential and its argument 4 e + |s - m| e more
      P         u of each weight (f16: 2^-25 absolute more, where P is subnormal;
                the row sum is at least 1 in P's unit)
      sums      n + 32 operations in O and in the row sum (parts merged in float32)
      O         u of the result
    """
    H, hd = q.shape[1], q.shape[2]
    page, Hkv = k_cache.shape[1], k_cache.shape[2]
    G = H // Hkv
    u, e = torch.finfo(q.dtype).eps / 2, 2.0 ** -23
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for r in range(len(kv_lens)):
        a, b, n = cu_q[r], cu_q[r + 1], kv_lens[r]
        if a == b or n <= 0:
            continue
        pages = table[r, : -(-n // page)].long()
        for g in range(Hkv):
            k = k_cache[pages, :, g].reshape(-1, hd)[:n].double()
            v = v_cache[pages, :, g].reshape(-1, hd)[:n].double()
            pos = positions[a:b].long()
            rows = torch.nonzero(pos >= 0).flatten()  # the others see nothing
            if rows.numel() == 0:
                continue
            hidden = torch.arange(n, device=q.device)[None, None, :] > pos[rows][:, None, None]
            qq = q[a:b, g * G:(g + 1) * G][rows].double()  # [rows, G, hd]
            s = (qq @ k.T) * scale
            # a masked score must not reach the result, whatever it is
            size = (qq.abs() @ k.abs().T).masked_fill(hidden, 0.0).amax(-1, keepdim=True) * scale
            low = s.masked_fill(hidden, math.inf).amin(-1, keepdim=True)
            s = s.masked_fill(hidden, -math.inf)
            spread = (s.amax(-1, keepdim=True) - low) / math.log(2)
            w = torch.softmax(s, -1)
            out = weighted(w, v, hidden)
            vis = torch.clamp(pos[rows] + 1, max=n)[:, None, None].double()
            rel = u + 2 * (hd + 4) * e * size + (8 + spread) * e + 2 * (vis + 32) * e
            t = rel * weighted(w, v.abs(), hidden) + u * out.abs()
            if q.dtype == torch.float16:
                t = t + 2.0 ** -25 * weighted((~hidden).double().expand_as(w), v.abs(), hidden)
            at = (a + rows)[:, None].expand(-1, G), torch.arange(g * G, (g + 1) * G, device=q.device).expand(len(rows), G)
            o[at], tol[at] = out, t
    return o, tol


def make_cache(kv_lens, page, Hkv, hd, dtype, gen, device, joint=False, spare=2, fill=None):
    """Random cache, table int32 [R,P] of shuffled pages (-1 behind a request's
    last). ``fill``: the value of every slot that no request holds."""
    need = [-(-n // page) for n in kv_lens]
    pages, width = sum(need) + spare, max(need + [1])
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(kv_lens), width), -1, dtype=torch.int32)
    at = 0
    for r, m in enumerate(need):
        table[r, :m] = torch.tensor(order[at:at + m], dtype=torch.int32)
        at += m
    kv = torch.randn((pages, 2, page, Hkv, hd), generator=gen).to(dtype)
    if fill is not None:
        held = torch.zeros((pages, page), dtype=torch.bool)
        for r, n in enumerate(kv_lens):
            for p in range(n):
                held[int(table[r, p // page]), p % page] = True
        kv.masked_fill_(~held[:, None, :, None, None], fill)
    kv = kv.to(device)
    if joint:
        return kv[:, 0], kv[:, 1], table.to(device)
    return kv[:, 0].contiguous(), kv[:, 1].contiguous(), table.to(device)
