"""Plain 64-bit statements of the paged 4-bit cache's operators, for the tests."""

import math

import torch


def quantise(x):
    """codes (int64), step, zero (bf16) of rows x [..., hd]: the definition, row by row."""
    x = x.float()
    zero = x.amin(-1).to(torch.bfloat16)
    span = x.amax(-1) - zero.float()
    # (on a GPU torch divides by a plain number as a product with its reciprocal)
    step = torch.where(span > 0, span / torch.full_like(span, 15.0), 0.0).to(torch.bfloat16)
    ok = torch.isfinite(x).all(-1) & torch.isfinite(zero.float()) & torch.isfinite(step.float())
    live = ok & (step > 0)
    q = (x.double() - zero.double()[..., None]) / torch.where(live, step, 1.0).double()[..., None]
    codes = torch.where(live[..., None], q.round().clamp(0, 15), 0.0).long()
    nan = torch.full_like(step, math.nan)
    return codes, torch.where(ok, step, nan), torch.where(ok, zero, nan)


def values(x):
    """What rows x read back as, fp64."""
    c, s, z = quantise(x)
    return z.double()[..., None] + c.double() * s.double()[..., None]


def empty_pool(pages, nkv, hd, page, fill=0, device="cpu"):
    return torch.full((pages, nkv, page * (hd + 8)), fill, dtype=torch.uint8, device=device)


def store(pool, hd, slots, k, v):
    """Rows k, v [n, nkv, hd] written to a pool (any device), by the layout's definition."""
    page = pool.shape[2] // (hd + 8)
    for i, x in enumerate((k, v)):
        c, s, z = quantise(x)
        codes = (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
        par = torch.stack([s, z], -1).view(torch.uint8)
        keep = (slots >= 0) & (slots < pool.shape[0] * page)
        at, off = slots[keep] // page, slots[keep] % page
        head = torch.arange(pool.shape[1], device=pool.device)[None, :, None]
        half = page * hd // 2
        col = torch.arange(hd // 2, device=pool.device)
        pool[at[:, None, None], head, off[:, None, None] * (hd // 2) + i * half + col] = codes[keep]
        col = torch.arange(4, device=pool.device)
        pool[at[:, None, None], head,
             off[:, None, None] * 4 + 2 * half + i * 4 * page + col] = par[keep]


def load(pool, hd):
    """(k, v) fp64 [pages, nkv, page, hd] of a whole pool."""
    page = pool.shape[2] // (hd + 8)
    half = page * hd // 2
    got = []
    for i in range(2):
        codes = pool[..., i * half:(i + 1) * half].reshape(*pool.shape[:2], page, hd // 2)
        par = pool[..., 2 * half + 4 * page * i:2 * half + 4 * page * (i + 1)].contiguous()
        par = par.view(torch.bfloat16).reshape(*pool.shape[:2], page, 2).double()
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
        got.append(par[..., 1:] + c * par[..., :1])
    return got


def attention(q, pool, table, lens, cu, scale, out, max_rows=None):
    """fp64 result rows written into a double copy of `out`, and per row the
    largest sum of |q_d k_td| * scale over what it sees (for error bounds)."""
    n, nq, hd = q.shape
    nkv, page = pool.shape[1], pool.shape[2] // (hd + 8)
    k_all, v_all = load(pool, hd)
    out = out.double().clone()
    size = torch.zeros(n, nq, dtype=torch.float64, device=q.device)
    for b in range(len(lens)):
        r0, r1 = max(0, cu[b]), min(n, cu[b + 1])
        rows = r1 - r0
        if rows <= 0 or (max_rows is not None and rows > max_rows):
            continue
        for i in range(rows):
            sees = max(0, min(lens[b] - rows + i + 1, table.shape[1] * page))
            pos = torch.arange(sees, device=q.device)
            pages = table[b][pos // page].long()
            fine = (pages >= 0) & (pages < pool.shape[0])
            pos, pages = pos[fine], pages[fine]
            if not len(pos):
                out[r0 + i] = 0
                continue
            k = k_all[pages, :, pos % page].transpose(0, 1).repeat_interleave(nq // nkv, 0)
            v = v_all[pages, :, pos % page].transpose(0, 1).repeat_interleave(nq // nkv, 0)
            x = q[r0 + i].double() * scale
            p = torch.softmax((k * x[:, None]).sum(-1), -1)
            out[r0 + i] = (p[..., None] * v).sum(1)
            size[r0 + i] = (k * x[:, None]).abs().sum(-1).amax(-1)
    return out, size


def plan(lens, joins, table, free, used, page, rows):
    """The definition, request by request. Lists in; a dict of lists out."""
    cu, slots, positions, after = [0], [-1] * rows, [-1] * rows, []
    asked = taken = joined = 0
    table = [list(t) for t in table]
    left = len(free) - used if 0 <= used <= len(free) else 0
    for b, (held, n) in enumerate(zip(lens, joins)):
        sane = held >= 0 and n >= 0
        n = max(0, n)
        joined += n
        have = -(-held // page) if sane else 0
        want = -(-(held + n) // page) if sane else 0
        ok = sane and joined <= rows and want <= len(table[b])
        if ok:
            asked += want - have
            ok = want == have or asked <= left
        if ok:
            for j in range(have, want):
                table[b][j] = free[used + asked - (want - j)]
            taken += want - have
        for r in range(cu[-1], min(joined, rows)):
            positions[r] = held + r - cu[-1]
            if ok:
                slots[r] = table[b][positions[r] // page] * page + positions[r] % page
        after.append(held + n if ok else held)
        cu.append(min(joined, rows))
    return dict(cu_rows=cu, lens=after, used=[used + taken], slots=slots, positions=positions,
                table=table)
