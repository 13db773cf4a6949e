"""The operators of the paged 4-bit KV cache: what is measured, in plain torch and through the framework.

  plan     block tables and slot maps from request lengths
  append   K/V rows quantised to 4 bits and stored through the slot map, and the values they stand for read back
  attend   attention over the paged 4-bit cache: one row per request, a few rows, prompt chunks

Layout of the cache: `pool` uint8 [pages, n_kv, page * (hd + 8)]; a block (one page of one kv head) holds the K codes
[page, hd / 2], the V codes [page, hd / 2], then K's and V's (step, zero) as bf16 [page, 2] each. Byte j of a code
row has element 2j in its low four bits and 2j + 1 in the high ones. A row stands for zero + code * step.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # every step of a small running batch: one new row for each of 8 requests
        dict(name="plan_step_8", op="plan", b=8, ctx=700, rows=1, page=16, short=False),
        # a scheduler's step on a busy server: 1024 requests, prompts of up to 96 rows among them
        dict(name="plan_mixed_1024", op="plan", b=1024, ctx=9000, rows=96, page=32, short=False),
        # one layer of one decode step of 16 sequences, fp32 activations as the engine has them
        dict(name="append_step_16", op="append", n=16, nkv=8, hd=128, page=16, type="float32", fused=True),
        # one layer of a long prompt batch, k and v as slices of the projection rows
        dict(name="append_prompt_16391", op="append", n=16391, nkv=8, hd=128, page=32, type="float32", fused=True),
        # the head size of the 1B workload, bf16 rows
        dict(name="append_bf16_4097", op="append", n=4097, nkv=8, hd=64, page=16, type="bfloat16", fused=False),
        # one request, the 0.6B workload's heads and its 512 cached positions
        dict(name="decode_1x513", op="attend", b=1, rows=1, ctx=513, nq=16, nkv=8, hd=128, page=16, type="float32"),
        # 16 sequences around 2048 positions, the 8B workload's batched decode, uneven lengths
        dict(name="decode_16x2048", op="attend", b=16, rows=1, ctx=2048, nq=32, nkv=8, hd=128, page=16, type="float32"),
        # a full server: 64 requests of up to 16384 positions, bf16
        dict(name="decode_64x16384_bf16", op="attend", b=64, rows=1, ctx=16384, nq=32, nkv=8, hd=128, page=32, type="bfloat16"),
        # one very long context, the 1B workload's heads
        dict(name="decode_1x131071", op="attend", b=1, rows=1, ctx=131071, nq=32, nkv=8, hd=64, page=64, type="float32"),
        # drafted tokens checked together: up to 4 rows for each of 8 requests, three query heads per kv head
        dict(name="verify_8x4_fp16", op="attend", b=8, rows=4, ctx=4099, nq=12, nkv=4, hd=64, page=16, type="float16"),
        # a fresh prompt, all rows at once
        dict(name="prompt_1x4096", op="attend", b=1, rows=4096, ctx=4096, nq=32, nkv=8, hd=128, page=32, type="float32"),
        # prompt chunks that join contexts already in the cache, a decoding request among them
        dict(name="chunks_4x1000_bf16", op="attend", b=4, rows=1000, ctx=8191, nq=16, nkv=8, hd=128, page=16, type="bfloat16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend"])
    page = rng.choice([16, 32, 64])
    if op == "plan":
        return dict(op=op, b=_log(rng, 1, 1024), ctx=_log(rng, 1, 9000), rows=_log(rng, 1, 96), page=page,
                    short=rng.random() < 0.25)
    dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
    hd = rng.choice([64, 128])
    if op == "append":
        return dict(op=op, n=_log(rng, 1, 16391), nkv=rng.choice([1, 2, 4, 8]), hd=hd, page=page, type=dtype,
                    fused=rng.random() < 0.5)
    nkv, group = rng.choice([(8, 2), (8, 4), (4, 3), (8, 1), (1, 8), (2, 5), (2, 16)])
    nq = nkv * group
    b = _log(rng, 1, 64)
    rows = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
    # a padded case holds at most as many cached values and scores as the largest listed ones
    ctx = min(131071, (1 << 30) // (b * nkv * hd), (1 << 29) // (b * nq * rows))
    rows = min(rows, max(1, ctx))
    return dict(op=op, b=b, rows=rows, ctx=_log(rng, min(rows, ctx), max(ctx, rows)), nq=nq, nkv=nkv, hd=hd, page=page, type=dtype)


def _spread(i, n):
    """A value in [0, n) for place i, uneven and the same for every seed."""
    return int(n * math.modf((i + 1) * 0.6180339887)[0])


def _requests(case):
    """(positions held before, rows that join) of every request; the first is the longest."""
    b, ctx, rows = case["b"], case["ctx"], case["rows"]
    held, new = [], []
    for i in range(b):
        n = rows if i == 0 else 1 + _spread(i, rows)
        if case["op"] == "attend" and rows > 8 and i % 4 == 3:
            n = 1               # a decoding request among the prompts
        if b >= 8 and i % 8 == 5:
            n = 0               # an idle place of the batch
        total = ctx if i == 0 else 1 + _spread(3 * i + 1, ctx)
        if case["op"] == "plan":
            held.append(total if i % 3 else 0)
        else:
            held.append(max(0, total - n))
        new.append(n)
    return held, new


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _quantise(x):
    """codes (uint8), step and zero (bf16) of rows x [..., hd]."""
    x = x.float()
    zero = x.amin(-1).to(torch.bfloat16)
    span = x.amax(-1) - zero.float()
    # a tensor of fifteens: by a plain number torch multiplies with its reciprocal
    step = torch.where(span > 0, span / torch.full_like(span, 15.0), torch.zeros_like(span)).to(torch.bfloat16)
    ok = torch.isfinite(x).all(-1) & torch.isfinite(step.float()) & torch.isfinite(zero.float())
    live = ok & (step.float() > 0)
    # 64 bits: whether a value lies above or below the middle of two codes
    safe = torch.where(live, step.double(), torch.ones_like(span, dtype=torch.float64))
    code = ((x.double() - zero.double().unsqueeze(-1)) / safe.unsqueeze(-1)).round().clamp(0, 15)
    code = torch.where(live.unsqueeze(-1), code, torch.zeros_like(code)).to(torch.uint8)
    nan = torch.full_like(step, float("nan"))
    return code, torch.where(ok, step, nan), torch.where(ok, zero, nan)


def _pack(code, step, zero):
    """bytes [..., hd / 2] of the codes and [..., 4] of (step, zero)."""
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack([step, zero], -1).view(torch.uint8)


def _split(blocks, page, hd):
    """K codes, V codes [..., page, hd / 2] and K, V (step, zero) [..., page, 2] of blocks [..., bytes]."""
    n, lead = page * hd // 2, blocks.shape[:-1]
    kc, vc = (blocks[..., i * n:(i + 1) * n].reshape(*lead, page, hd // 2) for i in (0, 1))
    kp, vp = (blocks[..., 2 * n + 4 * i * page:2 * n + 4 * (i + 1) * page].contiguous().view(torch.bfloat16)
              .reshape(*lead, page, 2) for i in (0, 1))
    return kc, vc, kp, vp


def _values(codes, params, dtype=torch.float32):
    """zero + code * step [..., hd]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(dtype)
    return c.mul_(params[..., 0:1].to(dtype)).add_(params[..., 1:2].to(dtype))


def _pool_of(k, v):
    """A packed pool of k, v [pages, n_kv, page, hd]."""
    parts = [_pack(*_quantise(x)) for x in (k, v)]
    return torch.cat([p[0].flatten(-2) for p in parts] + [p[1].flatten(-2) for p in parts], -1)


def _prepare_plan(case, g):
    held, new = _requests(case)
    page = case["page"]
    want = [-(-(h + n) // page) for h, n in zip(held, new)]
    have = [-(-h // page) for h in held]
    total, need = sum(have), sum(want) - sum(have)
    width = max(want)
    pages = total + need + 5
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    # the pages that the requests hold already are the first of the order; the rest are free
    col = torch.arange(width, device=DEV)
    lens = torch.tensor(held, dtype=torch.int64, device=DEV)
    n_have = (lens + page - 1) // page
    start = torch.cumsum(n_have, 0) - n_have
    at = (start.unsqueeze(1) + col).clamp(max=max(total - 1, 0))
    table = torch.where(col < n_have.unsqueeze(1), order[at], torch.full_like(order[at], -1))
    # `short`: the free pages do not last for all requests
    free = order[total:total + (need // 2 if case["short"] else need + 5)].contiguous()
    rows = sum(new) + 3
    return dict(lens=lens, new=torch.tensor(new, dtype=torch.int64, device=DEV), table=table.contiguous(),
                free=free, used=torch.zeros(1, dtype=torch.int64, device=DEV), page=page, rows=rows)


def _prepare_append(case, g):
    n, nkv, hd, page = case["n"], case["nkv"], case["hd"], case["page"]
    dtype = TYPES[case["type"]]
    pages = -(-n // page) + 2
    # keys after their rotation have channels of very different size, and offsets
    size = torch.exp(0.7 * torch.randn(nkv, hd, generator=g, device=DEV))
    shift = 2.0 * torch.randn(nkv, hd, generator=g, device=DEV) * (torch.rand(nkv, hd, generator=g, device=DEV) < 0.05)
    k = torch.randn(n, nkv, hd, generator=g, device=DEV) * size + shift
    v = torch.randn(n, nkv, hd, generator=g, device=DEV)
    if case["fused"]:
        # slices of the projection rows: q heads, k heads, v heads side by side
        rows = torch.zeros(n, 4 * nkv, hd, dtype=dtype, device=DEV)
        rows[:, 2 * nkv:3 * nkv] = k.to(dtype)
        rows[:, 3 * nkv:] = v.to(dtype)
        k, v = rows[:, 2 * nkv:3 * nkv], rows[:, 3 * nkv:]
    else:
        k, v = k.to(dtype), v.to(dtype)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:n].clone()
    if n > 8:
        slots[n // 2] = -1       # a row that is not stored
    pool = torch.zeros(pages, nkv, page * (hd + 8), dtype=torch.uint8, device=DEV)
    return dict(k=k, v=v, slots=slots, pool=pool, page=page, hd=hd)


def _prepare_attend(case, g):
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    dtype = TYPES[case["type"]]
    held, new = _requests(case)
    total = [h + n for h, n in zip(held, new)]
    width = -(-max(total) // page)
    count = [-(-t // page) for t in total]
    pages = sum(count) + 1
    size = torch.exp(0.5 * torch.randn(nkv, 1, hd, generator=g, device=DEV))
    size = size / size.square().mean(-1, keepdim=True).sqrt()
    pool = torch.empty(pages, nkv, page * (hd + 8), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 27) // (nkv * page * hd))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        k = torch.randn(n, nkv, page, hd, generator=g, device=DEV) * size
        v = torch.randn(n, nkv, page, hd, generator=g, device=DEV)
        pool[at:at + n] = _pool_of(k, v)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    c = torch.tensor(count, device=DEV)
    start = torch.cumsum(c, 0) - c
    col = torch.arange(width, device=DEV)
    at = (start.unsqueeze(1) + col).clamp(max=pages - 1)
    table = torch.where(col < c.unsqueeze(1), order[at], torch.zeros_like(order[at])).contiguous()
    rows = sum(new)
    q = torch.randn(rows + 2, nq, hd, generator=g, device=DEV) * 1.5    # two rows behind the last request
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int64, device=DEV)
    return dict(q=q.to(dtype), pool=pool, table=table, lens=torch.tensor(total, dtype=torch.int64, device=DEV),
                cu=cu, rows=case["rows"], n=rows, out=torch.full((rows + 2, nq, hd), 2.0 ** -8, dtype=dtype, device=DEV),
                scale=hd ** -0.5, page=page, nkv=nkv, hd=hd)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(plan=_prepare_plan, append=_prepare_append, attend=_prepare_attend)[case["op"]](case, g)
    state["op"] = case["op"]
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _plan_plain(s):
    lens, new, table, free, page, rows = s["lens"], s["new"], s["table"], s["free"], s["page"], s["rows"]
    width = table.shape[1]
    cu_in = torch.cumsum(new, 0)
    have, want = (lens + page - 1) // page, (lens + new + page - 1) // page
    fits = (cu_in <= rows) & (want <= width)
    need = torch.where(fits, want - have, torch.zeros_like(have))
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (s["used"] + upto <= free.numel()))
    taken = torch.where(granted, need, torch.zeros_like(need))
    col = torch.arange(width, device=lens.device)
    j = col - have.unsqueeze(1)
    fresh = (j >= 0) & (j < taken.unsqueeze(1))
    if free.numel():
        at = (s["used"] + (upto - need).unsqueeze(1) + j).clamp(0, free.numel() - 1)
        table.copy_(torch.where(fresh, free[at], table))
    cu = torch.cat([torch.zeros_like(cu_in[:1]), cu_in.clamp(max=rows)])
    r = torch.arange(rows, device=lens.device)
    b = torch.searchsorted(cu[1:].contiguous(), r, right=True)
    live = b < lens.numel()
    b = b.clamp(max=lens.numel() - 1)
    pos = lens[b] + r - cu[b]
    entry = table[b, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where(live & granted[b], entry * page + pos % page, torch.full_like(pos, -1))
    return dict(cu_rows=cu, lens=torch.where(granted, lens + new, lens), used=s["used"] + taken.sum(),
                slots=slots, positions=torch.where(live, pos, torch.full_like(pos, -1)), table=table)


def _append_plain(s):
    pool, slots, page, hd = s["pool"], s["slots"], s["page"], s["hd"]
    n = page * hd // 2
    live = slots >= 0
    at, off = torch.where(live, slots, torch.zeros_like(slots)) // page, slots % page
    nkv = pool.shape[1]
    head = torch.arange(nkv, device=pool.device)
    # rows that are not stored go to a page of their own behind the pool
    at = torch.where(live, at, torch.full_like(at, pool.shape[0]))
    more = torch.cat([pool, torch.zeros_like(pool[:1])])
    got = []
    for i, x in enumerate((s["k"], s["v"])):
        codes, params = _pack(*_quantise(x))
        c = off.view(-1, 1, 1) * (hd // 2) + i * n + torch.arange(hd // 2, device=pool.device)
        p = off.view(-1, 1, 1) * 4 + 2 * n + 4 * i * page + torch.arange(4, device=pool.device)
        a, h = at.view(-1, 1, 1), head.view(1, -1, 1)
        more[a, h, c] = codes
        more[a, h, p] = params
        back = _values(more[a, h, c], more[a, h, p].view(torch.bfloat16))
        got.append(torch.where(live.view(-1, 1, 1), back, torch.zeros_like(back)))
    pool.copy_(more[:-1])
    return got


def _attend_plain(s):
    q, pool, table, lens, cu, page, nkv, hd = (s[x] for x in ("q", "pool", "table", "lens", "cu", "page", "nkv", "hd"))
    b, rows, nq = lens.numel(), s["rows"], q.shape[1]
    kc, vc, kp, vp = _split(pool[table.long()], page, hd)      # [b, width, nkv, page, ...]
    order = (0, 2, 1, 3, 4)
    t = table.shape[1] * page
    n = cu[1:] - cu[:-1]
    i = torch.arange(rows, device=q.device)
    at = (cu[:-1].unsqueeze(1) + i)
    live = i < n.unsqueeze(1)
    qb = q[torch.where(live, at, torch.zeros_like(at))].float()            # [b, rows, nq, hd]
    qb = qb.view(b, rows, nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4).reshape(b, nkv, -1, hd)
    k = _values(kc, kp).permute(order).reshape(b, nkv, t, hd)
    score = torch.matmul(qb, k.transpose(-1, -2)).mul_(s["scale"])
    del k
    sees = (lens - n).unsqueeze(1) + i + 1                                   # positions below this one
    hide = torch.arange(t, device=q.device) >= torch.minimum(sees, lens.unsqueeze(1)).unsqueeze(-1)
    score = score.view(b, nkv, -1, rows, t).masked_fill_(hide.view(b, 1, 1, rows, t), -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = score.sum(-1, keepdim=True)
    v = _values(vc, vp).permute(order).reshape(b, nkv, t, hd)
    v = torch.where((torch.arange(t, device=q.device) < lens.unsqueeze(1)).view(b, 1, t, 1), v, torch.zeros_like(v))
    o = torch.matmul(score.view(b, nkv, -1, t), v).view(b, nkv, -1, rows, hd)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 3, 1, 2, 4).reshape(b * rows, nq, hd).to(q.dtype)
    # rows that no request has go to a row of their own behind the output
    out = torch.cat([s["out"], torch.zeros_like(s["out"][:1])])
    out[torch.where(live, at, torch.full_like(at, q.shape[0])).view(-1)] = o
    s["out"].copy_(out[:-1])
    return s["out"]


def run(state):
    if own:
        from quartz_b200 import device as qd
        if state["op"] == "plan":
            p = qd.kv4_plan(state["lens"], state["new"], state["table"], state["free"], state["used"],
                            page_size=state["page"], rows=state["rows"])
            return dict(cu_rows=p.cu_rows, lens=p.lens, used=p.used, slots=p.slots, positions=p.positions,
                        table=state["table"])
        if state["op"] == "append":
            qd.kv4_append(state["k"], state["v"], state["pool"], state["slots"])
            return list(qd.kv4_gather(state["pool"], state["slots"], state["hd"]))
        return qd.kv4_attention(state["q"], state["pool"], state["table"], state["lens"], cu_rows=state["cu"],
                                max_rows=state["rows"], scale=state["scale"], out=state["out"])
    return dict(plan=_plan_plain, append=_append_plain, attend=_attend_plain)[state["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "append":
        size = TYPES[case["type"]].itemsize
        values = 2 * case["n"] * case["nkv"] * case["hd"]
        packed = 2 * case["n"] * case["nkv"] * (case["hd"] // 2 + 4)
        # rows in, codes out; codes in, values out
        return {"bytes": values * size + 2 * packed + 4 * values + 16 * case["n"], "flops": 6 * values}
    held, new = _requests(case)
    if case["op"] == "plan":
        page = case["page"]
        fresh = sum(-(-(h + n) // page) - -(-h // page) for h, n in zip(held, new))
        return {"bytes": 32 * case["b"] + 16 * sum(new) + 8 * fresh, "flops": 4 * case["b"] + 4 * sum(new)}
    size, nq, nkv, hd = TYPES[case["type"]].itemsize, case["nq"], case["nkv"], case["hd"]
    cached = sum(h + n for h, n in zip(held, new) if n) * nkv * (hd + 8)
    seen = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))
    return {"bytes": cached + 2 * sum(new) * nq * hd * size, "flops": 4 * hd * nq * seen}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_plan(s):
    lens, new, free = s["lens"].tolist(), s["new"].tolist(), s["free"].tolist()
    table, used, page, rows = s["table"].tolist(), int(s["used"]), s["page"], s["rows"]
    cu, slots, positions, after, asked = [0], [-1] * rows, [-1] * rows, [], 0
    taken, joined = 0, 0
    for b, (held, n) in enumerate(zip(lens, new)):
        have, want = math.ceil(held / page), math.ceil((held + n) / page)
        joined += n
        fits = joined <= rows and want <= len(table[b])
        if fits:
            asked += want - have
        ok = fits and (want == have or used + asked <= len(free))
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
    as_long = lambda x: torch.tensor(x, dtype=torch.int64)  # noqa: E731
    return dict(cu_rows=as_long(cu), lens=as_long(after), used=as_long([used + taken]), slots=as_long(slots),
                positions=as_long(positions), table=torch.tensor(table, dtype=torch.int32))


def _exact_append(s):
    got = []
    for x in (s["k"], s["v"]):
        x = x.double()
        # the zero and the step are what is kept: 16-bit values, chosen in 32 bits
        zero = x.min(-1, keepdim=True).values.bfloat16().double()
        reach = (x.max(-1, keepdim=True).values - zero).float()
        fifteen = torch.full_like(reach, 15, dtype=torch.float64)
        step = (reach.clamp(min=0).double() / fifteen).float().bfloat16().double()
        code = torch.clamp(torch.round((x - zero) / torch.where(step > 0, step, 1.0)), 0, 15) * (step > 0)
        back = zero + code * step
        back[s["slots"] < 0] = 0
        got.append(back)
    return got


def _exact_attend(s):
    page, hd, nkv = s["page"], s["hd"], s["nkv"]
    out, lens, cu = s["out"].double(), s["lens"].tolist(), s["cu"].tolist()
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if not n:
            continue
        blocks = s["pool"][s["table"][b, :math.ceil(length / page)].long()]          # [pages, nkv, bytes]
        q = s["q"][cu[b]:cu[b + 1]].double() * s["scale"]
        half = page * hd // 2
        for h in range(nkv):
            def rows(at, par):
                raw = blocks[:, h, at:at + half].reshape(-1, hd // 2)
                code = torch.empty(raw.shape[0], hd, dtype=torch.float64, device=raw.device)
                code[:, ::2], code[:, 1::2] = raw % 16, raw // 16
                sz = blocks[:, h, par:par + 4 * page].contiguous().view(torch.bfloat16).reshape(-1, 2).double()
                return (code * sz[:, :1] + sz[:, 1:])[:length]
            k, v = rows(0, 2 * half), rows(half, 2 * half + 4 * page)
            group = q.shape[1] // nkv
            for at in range(0, n, 512):
                i = torch.arange(at, min(n, at + 512), device=k.device)
                see = torch.arange(length, device=k.device) <= (length - n + i).unsqueeze(1)
                score = torch.einsum("igd,td->igt", q[i, h * group:(h + 1) * group], k)
                p = torch.softmax(score.masked_fill(~see.unsqueeze(1), -math.inf), -1)
                out[cu[b] + i, h * group:(h + 1) * group] = torch.einsum("igt,td->igd", p, v)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return dict(plan=_exact_plan, append=_exact_append, attend=_exact_attend)[case["op"]](s)
