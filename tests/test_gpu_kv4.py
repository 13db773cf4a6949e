"""The paged 4-bit KV cache on the GPU against plain 64-bit statements (tests/_kv4.py).

What is integer (plans, codes, parameters) has to be equal; read-back values
are one fp32 rounding of z + c * s. Attention's bound: q is split into two fp16
values (2^-23 of the row's largest), the scores accumulate hd / 16 * 2 times in
fp32 with truncation (2^-23 each) over unsigned codes, whose sums are at most
about four times sum |q k|; so a score is off by at most
4 A (hd / 16 + 8) 2^-23 with A = scale * sum |q k|, a weight by that relatively
plus 2^-21 of exponent and split, and a result by twice it times max |v| (the
normalisation has the same error), plus the rounding to the output's type. For
many rows of a 16-bit type the weights are single fp16 values: each is off by at
most 2^-11 of itself, and multiplies a value of at most 16 steps of its row, so
the result by at most 2^-11 * 16 s <= 2^-11 * 2.2 max |v| (16 / 15 of the row's
range, which is at most 2 max |v|) more.
"""

import math
import random

import pytest

from tests import _kv4 as P

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _dev():
    from quartz_b200 import device as qd
    return qd, torch.device("cuda", 0)


def _i64(x, dev):
    return torch.tensor(x, dtype=torch.int64, device=dev)


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------

def _run_plan(lens, joins, table, free, used, page, rows, in_place=False):
    qd, dev = _dev()
    tl, tj = _i64(lens, dev), _i64(joins, dev)
    tt = torch.tensor(table, dtype=torch.int32, device=dev)
    tf = torch.tensor(free, dtype=torch.int32, device=dev)
    tu = _i64([used], dev)
    p = qd.kv4_plan(tl, tj, tt, tf, tu, page, rows, lens_out=tl if in_place else None,
                    used_out=tu if in_place else None)
    if in_place:
        assert p.lens is tl and p.used is tu
    else:
        assert tl.tolist() == list(lens) and tu.tolist() == [used]
    return dict(cu_rows=p.cu_rows.tolist(), lens=p.lens.tolist(), used=p.used.tolist(),
                slots=p.slots.tolist(), positions=p.positions.tolist(), table=tt.tolist())


@pytest.mark.parametrize("B,page,most", [(1, 16, 1), (7, 16, 40), (64, 32, 1), (300, 64, 9),
                                         (1025, 256, 3), (4096, 16, 2), (40, 128, 700)])
@pytest.mark.parametrize("short", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(B, page, most, short, in_place):
    rng = random.Random(B * 7 + page + short)
    lens = [rng.choice([0, 1, page - 1, page, page + 1, rng.randrange(5 * page)]) for _ in range(B)]
    joins = [rng.choice([0, 1, most, rng.randrange(most + 1)]) for _ in range(B)]
    width = max(-(-(h + n) // page) for h, n in zip(lens, joins)) or 1
    if short:
        width = max(1, width - 1)          # some requests outgrow the table
    need = sum(-(-(h + n) // page) - -(-h // page) for h, n in zip(lens, joins))
    free = rng.sample(range(10 * (need + 9)), need + 3)
    used = 2
    if short:
        free = free[:2 + need // 2]
    table = [[rng.randrange(1000) for _ in range(width)] for _ in range(B)]
    rows = sum(joins) + (0 if short else 5)
    got = _run_plan(lens, joins, table, free, used, page, rows, in_place)
    want = P.plan(lens, joins, table, free, used, page, rows)
    assert got == want


@pytest.mark.parametrize("case", [
    dict(lens=[3, 5], joins=[4, 4], rows=6),                 # the second request's rows do not fit
    dict(lens=[3, 5, 2], joins=[4, 9, 1], rows=6),           # ... nor those of requests behind it
    dict(lens=[-1, 5], joins=[1, 1], rows=4),                # negative length
    dict(lens=[3, 5], joins=[-7, 1], rows=4),                # negative row count
    dict(lens=[48, 0], joins=[1, 48], rows=64),              # the table's width
    dict(lens=[1 << 40, 0], joins=[1, 1], rows=4),           # a length no table holds
    dict(lens=[16, 16], joins=[0, 0], rows=0),               # nothing joins
    dict(lens=[0, 0], joins=[1, 1], rows=2, used=-1),        # a cursor outside the list
    dict(lens=[0, 16], joins=[1, 0], rows=2, used=99),
    dict(lens=[0, 1], joins=[1, 1], rows=2, free=[]),        # no free pages; the second needs none
])
def test_plan_refuses(case):
    case = dict(dict(free=[9, 8, 7, 6], used=0), **case)
    table = [[100 + 10 * b + j for j in range(3)] for b in range(len(case["lens"]))]
    args = (case["lens"], case["joins"], table, case["free"], case["used"], 16, case["rows"])
    assert _run_plan(*args) == P.plan(*args)


# ---------------------------------------------------------------------------
# append and gather
# ---------------------------------------------------------------------------

def _rows(n, nkv, hd, dtype, g, dev, layout="plain"):
    """k, v [n, nkv, hd] in one of several memory layouts."""
    def fill():
        x = torch.randn(n, nkv, hd, generator=g, device=dev)
        return (x * torch.exp(torch.randn(n, nkv, 1, generator=g, device=dev)) +
                torch.randn(n, nkv, 1, generator=g, device=dev)).to(dtype)
    k, v = fill(), fill()
    if layout == "slices":              # parts of projection rows
        wide = torch.zeros(n, 4 * nkv, hd, dtype=dtype, device=dev)
        wide[:, 2 * nkv:3 * nkv], wide[:, 3 * nkv:] = k, v
        return wide[:, 2 * nkv:3 * nkv], wide[:, 3 * nkv:]
    if layout == "odd":                 # rows that start off any 16-byte boundary
        wide = torch.zeros(2, n, nkv, hd + 1, dtype=dtype, device=dev)
        wide[0, ..., 1:], wide[1, ..., 1:] = k, v
        return wide[0, ..., 1:], wide[1, ..., 1:]
    if layout == "heads":               # heads outermost
        return (k.transpose(0, 1).contiguous().transpose(0, 1),
                v.transpose(0, 1).contiguous().transpose(0, 1))
    return k, v


def _check_append(k, v, page, pages, slots, fill=0xA5):
    """Append, compare every byte of the pool, then read back."""
    qd, dev = _dev()
    hd, nkv = k.shape[2], k.shape[1]
    pool = P.empty_pool(pages, nkv, hd, page, fill, dev)
    want = pool.clone()
    qd.kv4_append(k, v, pool, slots)
    P.store(want, hd, slots, k, v)
    half = page * hd // 2
    # parameters of NaN rows: any NaN
    wp, gp = (x[..., 2 * half:].contiguous().view(torch.bfloat16) for x in (want, pool))
    assert torch.equal(torch.isnan(wp), torch.isnan(gp))
    assert torch.equal(torch.nan_to_num(wp), torch.nan_to_num(gp))
    assert torch.equal(want[..., :2 * half], pool[..., :2 * half])
    gk, gv = qd.kv4_gather(pool, slots, hd)
    keep = ((slots >= 0) & (slots < pages * page))[:, None, None]
    for got, x in ((gk, k), (gv, v)):
        ref = torch.where(keep, P.values(x), 0.0)
        assert torch.equal(torch.isnan(ref), torch.isnan(got))
        # z + c * s rounded once to fp32
        assert torch.equal(torch.nan_to_num(ref).float(), torch.nan_to_num(got))
    return pool


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,nkv,page,layout", [
    (1, 1, 16, "plain"), (3, 8, 16, "slices"), (33, 3, 32, "odd"), (257, 2, 64, "heads"),
    (1000, 5, 128, "slices"), (70, 1, 256, "plain")])
def test_append_and_gather(dtype, hd, n, nkv, page, layout):
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(n + hd)
    k, v = _rows(n, nkv, hd, DTYPES[dtype], g, dev, layout)
    pages = n // page + 2
    slots = torch.randperm(pages * page, generator=g, device=dev)[:n].clone()
    if n > 2:
        slots[1] = -1
        slots[2] = pages * page           # one behind the pool
    _check_append(k, v, page, pages, slots)


@pytest.mark.parametrize("hd", [64, 128])
def test_append_border_values(hd):
    """Rows at the quantiser's edges: constants, zeros, ties between codes, one
    outlier, subnormal and huge ranges, and non-finite values in each place."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(5)
    base = torch.randn(hd, generator=g, device=dev)
    ties = (torch.arange(hd, device=dev) % 31).float() * 0.5          # z = 0, s = 1: halves tie
    ladder = torch.full((hd,), -8.0, device=dev)
    ladder[1:] = (torch.arange(hd - 1, device=dev) % 31) * 0.25 - 8.0
    rows = [torch.zeros(hd, device=dev), torch.full((hd,), 3.3, device=dev), ties, -ties, ladder,
            base * 1e-38, base * 1e-42, base * 1e-30, base * 1e38, base * 3e37, base + 1e6,
            base * 1e-3 + 100.0, torch.full((hd,), -1e-45, device=dev)]
    spike = base * 1e-3
    spike[hd // 2] = 1e4
    rows.append(spike)
    for bad in (math.nan, math.inf, -math.inf):
        for at in (0, 15, hd - 1):
            r = base.clone()
            r[at] = bad
            rows.append(r)
    both = base.clone()
    both[0], both[1] = 3.3e38, -3.3e38                                 # a range beyond fp32
    rows.append(both)
    # values one step to either side of the middle between two codes
    s = torch.tensor(0.37, device=dev).bfloat16().float()
    mids = (torch.arange(hd, device=dev) % 15 + 0.5) * s
    mids[0], mids[1] = 0.0, 15 * s
    for step in (0, 1, -1):
        m = mids.clone()
        m[2:] = torch.nextafter(m[2:], torch.full_like(m[2:], math.inf * step if step else 0)) if step else m[2:]
        rows.append(m)
    x = torch.stack(rows)
    k = x[:, None].contiguous()
    v = x.flip(0)[:, None].contiguous()
    pages = -(-len(rows) // 16) + 1
    _check_append(k, v, 16, pages, torch.arange(len(rows), device=dev))


def test_append_to_a_pool_beyond_32_bits():
    """Slots whose bytes lie past 4 GB."""
    qd, dev = _dev()
    if torch.cuda.mem_get_info(0)[0] < 8 << 30:
        pytest.skip("needs 8 GB of device memory")
    nkv, hd, page = 8, 128, 256
    block = nkv * page * (hd + 8)
    pages = (5 << 30) // block
    pool = torch.zeros(pages, nkv, page * (hd + 8), dtype=torch.uint8, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    k, v = _rows(40, nkv, hd, torch.float32, g, dev)
    slots = torch.arange(40, device=dev) + pages * page - 40
    qd.kv4_append(k, v, pool, slots)
    gk, gv = qd.kv4_gather(pool, slots, hd)
    assert torch.equal(gk, P.values(k).float()) and torch.equal(gv, P.values(v).float())
    assert not pool[:pages - 1].any()
    # and attention over the same pages
    table = torch.full((1, 1), pages - 1, dtype=torch.int32, device=dev)
    small = pool[pages - 1:].clone()
    q = torch.randn(1, nkv, hd, generator=g, device=dev)
    # the 40 rows are the page's last, so the context is the whole page
    out = qd.kv4_attention(q, pool, table, _i64([page], dev))
    ref = qd.kv4_attention(q, small, torch.zeros_like(table), _i64([page], dev))
    assert torch.equal(out, ref)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _context(lens, nkv, hd, page, g, dev, extra=2, width=None, k_scale=1.0, v_scale=1.0):
    """A pool with random rows for every position of every request, pages in a
    shuffled order; whatever no request holds is filled with NaN parameters."""
    count = [-(-max(0, t) // page) for t in lens]
    width = width or max(1, max(count))
    pages = sum(count) + extra
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    pool = P.empty_pool(pages, nkv, hd, page, 0xFF, dev)      # bf16 0xFFFF: NaN
    at = 0
    for b, t in enumerate(lens):
        own = order[at:at + count[b]]
        at += count[b]
        table[b, :min(width, count[b])] = own[:width]
        if t <= 0:
            continue
        pos = torch.arange(t, device=dev)
        slots = own[pos // page].long() * page + pos % page
        k = torch.randn(t, nkv, hd, generator=g, device=dev) * k_scale
        v = torch.randn(t, nkv, hd, generator=g, device=dev) * v_scale
        P.store(pool, hd, slots, k, v)
    return pool, table


def _check_attention(q, pool, table, lens, cu, scale=None, max_rows=1, out=None, **kw):
    qd, dev = _dev()
    hd = q.shape[2]
    s = hd ** -0.5 if scale is None else scale
    if out is None:
        out = torch.full_like(q, 0.25, memory_format=torch.contiguous_format)
    ref, size = P.attention(q, pool, table, lens, cu if cu is not None else list(range(len(lens) + 1)),
                            s, out, max_rows)
    got = qd.kv4_attention(q, pool, table, _i64(lens, dev),
                           cu_rows=None if cu is None else _i64(cu, dev), max_rows=max_rows,
                           scale=scale, out=out, **kw)
    assert got is out
    assert torch.equal(torch.isnan(ref), torch.isnan(got.double()))
    vmax = torch.nan_to_num(torch.stack(P.load(pool, hd))[1], nan=0.0).abs().max().item() or 1.0
    bound = vmax * (2 * 4 * size * (hd / 16 + 8) * 2.0 ** -23 + 2.0 ** -19)
    if q.dtype != torch.float32 and max_rows > 1:
        bound = bound + vmax * 2.2 * 2.0 ** -11
    bound = bound[..., None] + ref.abs() * torch.finfo(q.dtype).eps / 2
    err = torch.nan_to_num((got.double() - ref).abs(), nan=0.0)
    worst = (err - torch.nan_to_num(bound, nan=math.inf)).max().item()
    assert worst <= 0, (worst, err.max().item())
    group = q.shape[1] // pool.shape[1]
    if cu is not None and max_rows * group > 64 and q.is_contiguous() and not kw:
        # With rows behind the last request's there is work for the tensor cores' tiles:
        # the other kernel, held to the same bound.
        more = len(lens) + -(-80 // pool.shape[1]) * 128 // group + 1
        wide = torch.full((q.shape[0] + more, *q.shape[1:]), 0.25, dtype=q.dtype, device=dev)
        wide_q = wide.clone()
        wide_q[:q.shape[0]] = q
        qd.kv4_attention(wide_q, pool, table, _i64(lens, dev), cu_rows=_i64(cu, dev), max_rows=max_rows,
                         scale=scale, out=wide)
        assert (wide[cu[-1]:] == 0.25).all()
        other = wide[:q.shape[0]].double()
        seen = slice(0, cu[-1])
        assert torch.equal(torch.isnan(ref[seen]), torch.isnan(other[seen]))
        err = torch.nan_to_num((other - ref).abs(), nan=0.0)
        assert (err - torch.nan_to_num(bound, nan=math.inf))[seen].max().item() <= 0
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (4, 2), (8, 2), (6, 2), (10, 2), (8, 1), (16, 1), (20, 1)])
def test_decode_heads(dtype, hd, nq, nkv):
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(nq * 10 + nkv)
    lens = [37, 1, 130]
    pool, table = _context(lens, nkv, hd, 16, g, dev)
    q = torch.randn(len(lens), nq, hd, generator=g, device=dev).to(DTYPES[dtype])
    _check_attention(q, pool, table, lens, None)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("lens", [[0], [1], [2], [15], [16], [17], [63], [64], [65], [127, 0, 129],
                                  [5000], [0, 0, 0], [1, 2000, 3, 0, 700, 16], list(range(70))])
def test_decode_lengths(page, lens):
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(page + len(lens))
    pool, table = _context(lens, 2, 64, page, g, dev)
    q = torch.randn(len(lens) + 2, 6, 64, generator=g, device=dev)      # two rows of no request
    _check_attention(q, pool, table, lens, None)


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_long(hd):
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(hd)
    lens = [70001, 3]
    pool, table = _context(lens, 1, hd, 64, g, dev)
    q = torch.randn(2, 4, hd, generator=g, device=dev) * 2
    _check_attention(q, pool, table, lens, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 128), (3, 1, 64), (8, 1, 128)])
@pytest.mark.parametrize("rows,lens", [
    ([2], [2]), ([3], [100]), ([1, 4, 0, 2], [50, 4, 9, 81]), ([5, 1], [3, 1]),   # more rows than positions
    ([33, 1, 70], [33, 200, 150]), ([130], [300]), ([0, 0], [4, 5])])
def test_rows(dtype, nq, nkv, hd, rows, lens):
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(sum(rows))
    pool, table = _context(lens, nkv, hd, 16, g, dev)
    cu = [sum(rows[:i]) for i in range(len(rows) + 1)]
    q = torch.randn(cu[-1] + 3, nq, hd, generator=g, device=dev).to(DTYPES[dtype])
    _check_attention(q, pool, table, lens, cu, max_rows=max(1, max(rows)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,nkv,page", [(2, 2, 16), (4, 2, 256), (3, 1, 32), (5, 1, 16), (8, 1, 64),
                                         (16, 1, 16), (48, 1, 16), (130, 1, 16)])
@pytest.mark.parametrize("rows,lens", [
    ([129], [129]), ([40, 0, 65, 1], [40, 7, 400, 300]), ([200, 34], [150, 1200])])
def test_prompts(dtype, hd, nq, nkv, page, rows, lens):
    """Whole prompts, chunks on top of a context, more rows than positions, decoding
    and idle requests among them; groups that do not divide a tile."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(sum(rows) + nq)
    pool, table = _context(lens, nkv, hd, page, g, dev)
    cu = [sum(rows[:i]) for i in range(len(rows) + 1)]
    q = torch.randn(cu[-1] + 3, nq, hd, generator=g, device=dev).to(DTYPES[dtype])
    _check_attention(q, pool, table, lens, cu, max_rows=max(rows))
    qd.check_status()


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_edges(hd):
    """Bad pages, a table that ends early, NaN and infinite rows, steps of very
    different size, sharp scores, strided rows, in a prompt."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(21)
    rows, t = 100, 300
    cu = [0, rows]

    def fresh(**kw):
        pool, table = _context([t], 2, hd, 16, g, dev, **kw)
        return pool, table, torch.randn(rows, 4, hd, generator=g, device=dev)

    pool, table, q = fresh()
    table[0, 3], table[0, 9], table[0, 18] = -1, pool.shape[0], 1 << 30
    _check_attention(q, pool, table, [t], cu, max_rows=rows)
    table[:] = -7
    assert (_check_attention(q, pool, table, [t], cu, max_rows=rows) == 0).all()
    pool, table, q = fresh(width=10)
    _check_attention(q, pool, table, [t], cu, max_rows=rows)
    # a NaN key at 250 and an infinite value at 290 of kv head 1
    pool, table, q = fresh()
    k, v = torch.randn(2, 2, 2, hd, generator=g, device=dev)
    k[0, 1, 0], v[1, 1, 0] = math.nan, math.inf
    slots = _i64([int(table[0, p // 16]) * 16 + p % 16 for p in (250, 290)], dev)
    qd.kv4_append(k, v, pool, slots)
    got = _check_attention(q, pool, table, [t], cu, max_rows=rows)
    assert torch.isnan(got).any(-1).sum() == 2 * 50
    # one query row with an infinity spoils itself only
    pool, table, q = fresh()
    q[37, 2, 5] = math.inf
    got = qd.kv4_attention(q, pool, table, _i64([t], dev), cu_rows=_i64(cu, dev), max_rows=rows)
    assert torch.isnan(got).any(-1).nonzero().tolist() == [[37, 2]]
    # steps from 1e-25 to 1e25 (rising, falling), scores that rise or fall by hundreds
    pos = torch.arange(t, device=dev)
    for flip in (False, True):
        pool, table, q = fresh()
        ex = torch.linspace(-25, 25, t, device=dev)
        ex = ex.flip(0) if flip else ex
        k = torch.randn(t, 2, hd, generator=g, device=dev)
        v = torch.randn(t, 2, hd, generator=g, device=dev) * torch.pow(10.0, ex)[:, None, None]
        P.store(pool, hd, table[0][pos // 16].long() * 16 + pos % 16, k, v)
        _check_attention(q, pool, table, [t], cu, max_rows=rows)
        ramp = (-1.0 if flip else 1.0) * pos.float()[:, None, None]
        v = torch.randn(t, 2, hd, generator=g, device=dev)
        P.store(pool, hd, table[0][pos // 16].long() * 16 + pos % 16, ramp.expand(t, 2, hd), v)
        q = torch.ones(rows, 4, hd, device=dev)
        q[:, 1] = 0.0
        _check_attention(q, pool, table, [t], cu, max_rows=rows)
    for layout in ("slices", "odd", "heads"):
        pool, table, _ = fresh()
        q, out = _rows(rows, 4, hd, torch.float32, g, dev, layout)
        out.fill_(0.25)
        got = _check_attention(q, pool, table, [t], cu, max_rows=rows, out=out)
        want = got.clone()
        assert torch.equal(qd.kv4_attention(q, pool, table, _i64([t], dev), cu_rows=_i64(cu, dev),
                                            max_rows=rows, out=q), want)
    qd.check_status()


def test_long_prompt_same_bits_and_graph():
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(22)
    lens, rows = [900, 1500, 40], [900, 300, 1]
    pool, table = _context(lens, 2, 128, 32, g, dev)
    cu = _i64([0, 900, 1200, 1201], dev)
    q = torch.randn(1201, 8, 128, generator=g, device=dev)
    tl = _i64(lens, dev)
    first = qd.kv4_attention(q, pool, table, tl, cu_rows=cu, max_rows=900)
    out = torch.zeros_like(q)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        qd.kv4_attention(q, pool, table, tl, cu_rows=cu, max_rows=900, out=out)
    for _ in range(3):
        out.zero_()
        gr.replay()
        assert torch.equal(out, first)
    # each request alone, and each row as a decode step, agree within rounding
    for b, (r0, n) in enumerate(((0, 900), (900, 300), (1200, 1))):
        alone = qd.kv4_attention(q[r0:r0 + n], pool, table[b:b + 1], tl[b:b + 1],
                                 cu_rows=_i64([0, n], dev), max_rows=n)
        assert (alone - first[r0:r0 + n]).abs().max() < 2e-5     # (another kernel, for its few tiles)
        for i in (0, n // 2, n - 1):
            one = qd.kv4_attention(q[r0 + i:r0 + i + 1], pool, table[b:b + 1], tl[b:b + 1] - n + i + 1)
            assert (one - first[r0 + i]).abs().max() < 2e-5
    qd.check_status()


def test_rows_beyond_max_rows_are_left():
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(2)
    pool, table = _context([20, 30], 2, 64, 16, g, dev)
    q = torch.randn(5, 4, 64, generator=g, device=dev)
    got = _check_attention(q, pool, table, [20, 30], [0, 4, 5], max_rows=3)
    assert (got[:4] == 0.25).all()


def test_lengths_beyond_the_table_and_bad_pages():
    """Positions past the table are not seen; entries outside the pool are not
    read (their positions count as unseen), also when all of a request's are bad."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(3)
    lens = [100, 100, 40, 100000]
    pool, table = _context([100, 100, 40, 96], 2, 64, 16, g, dev, width=6)
    table[1, 2] = pool.shape[0]
    table[1, 4] = -5
    table[2] = 1 << 30
    q = torch.randn(4, 4, 64, generator=g, device=dev)
    got = _check_attention(q, pool, table, lens, None)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("k_scale,v_scale", [(1e-3, 1e-6), (1e-20, 1e20), (1.0, 1e-36), (8.0, 1.0),
                                             (1e-8, 1e30)])
def test_value_ranges(k_scale, v_scale):
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(4)
    lens = [90, 33]
    pool, table = _context(lens, 2, 64, 16, g, dev, k_scale=k_scale, v_scale=v_scale)
    q = torch.randn(2, 4, 64, generator=g, device=dev) * min(1e6, 1.0 / k_scale)
    _check_attention(q, pool, table, lens, None)


def test_steps_of_very_different_size():
    """V rows from 1e-25 to 1e25 in one context, in rising and falling order: the
    weights' exponent has to follow."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(6)
    for flip in (False, True):
        t, hd = 200, 64
        pool, table = _context([t], 1, hd, 16, g, dev)
        ex = torch.linspace(-25, 25, t, device=dev)
        v = torch.randn(t, 1, hd, generator=g, device=dev) * torch.pow(10.0, ex.flip(0) if flip else ex)[:, None, None]
        k = torch.randn(t, 1, hd, generator=g, device=dev)
        pos = torch.arange(t, device=dev)
        P.store(pool, hd, table[0][pos // 16].long() * 16 + pos % 16, k, v)
        _check_attention(torch.randn(1, 4, hd, generator=g, device=dev), pool, table, [t], None)


def test_sharp_and_equal_scores():
    """Scores that grow along the context by hundreds, fall by hundreds, and are all equal."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(7)
    t, hd = 300, 64
    for slope in (1.0, -1.0, 0.0):
        pool, table = _context([t], 1, hd, 16, g, dev)
        ramp = slope * torch.arange(t, device=dev).float()[:, None, None]
        k = ramp.expand(t, 1, hd).contiguous()
        v = torch.randn(t, 1, hd, generator=g, device=dev)
        pos = torch.arange(t, device=dev)
        P.store(pool, hd, table[0][pos // 16].long() * 16 + pos % 16, k, v)
        q = torch.ones(1, 2, hd, device=dev)
        q[0, 1] = 0.0                                   # a query of zeros: the mean of V
        _check_attention(q, pool, table, [t], None)


def test_non_finite_rows_stay_where_they_are_seen():
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(8)
    hd, lens = 64, [40, 40, 40, 40]
    pool, table = _context(lens, 2, hd, 16, g, dev)
    k = torch.randn(3, 2, hd, generator=g, device=dev)
    v = torch.randn(3, 2, hd, generator=g, device=dev)
    k[0, 0, 3] = math.nan                               # request 0, kv head 0: K
    v[1, 1, 5] = math.inf                               # request 1, kv head 1: V
    k[2], v[2] = math.nan, math.nan                     # request 2, past its length
    slot = lambda b, p: int(table[b, p // 16]) * 16 + p % 16  # noqa: E731
    qd.kv4_append(k, v, pool, _i64([slot(0, 7), slot(1, 39), slot(2, 39)], dev))
    q = torch.randn(4, 4, hd, generator=g, device=dev)
    q[3, 1, 0] = math.inf
    lens = [40, 40, 39, 40]
    got = _check_attention(q[:3], pool, table[:3], lens[:3], None)
    nan = torch.isnan(got).all(-1)
    assert nan.tolist() == [[True, True, False, False], [False, False, True, True], [False] * 4]
    got = qd.kv4_attention(q, pool, table, _i64(lens, dev))
    assert torch.isnan(got[3, 1]).all() and torch.isfinite(got[3, [0, 2, 3]]).all()


@pytest.mark.parametrize("layout", ["slices", "odd", "heads"])
def test_strided_queries_and_outputs(layout):
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(9)
    lens = [70, 9, 0]
    pool, table = _context(lens, 2, 128, 32, g, dev)
    q, out = _rows(3, 4, 128, torch.float32, g, dev, layout)
    out.fill_(0.25)
    got = _check_attention(q, pool, table, lens, None, out=out)
    # in place
    want = got.clone()
    again = qd.kv4_attention(q, pool, table, _i64(lens, dev), out=q)
    assert again is q and torch.equal(q, want)
    # one query row for all requests (stride 0)
    one = torch.randn(1, 4, 128, generator=g, device=dev)
    _check_attention(one.expand(3, 4, 128), pool, table, lens, None)


def test_same_bits_every_time():
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(10)
    lens = [3000, 1, 900, 64] * 8
    pool, table = _context(lens, 2, 128, 16, g, dev)
    q = torch.randn(len(lens), 8, 128, generator=g, device=dev)
    first = qd.kv4_attention(q, pool, table, _i64(lens, dev))
    for _ in range(5):
        assert torch.equal(first, qd.kv4_attention(q, pool, table, _i64(lens, dev)))


def test_other_streams_and_graphs_side_by_side():
    """Two captured graphs and an eager stream run the same context at once; each
    has its own workspace."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(11)
    lens = [4000, 77, 2500]
    pool, table = _context(lens, 2, 64, 16, g, dev)
    tl = _i64(lens, dev)
    qs = [torch.randn(3, 8, 64, generator=g, device=dev) for _ in range(3)]
    want = [qd.kv4_attention(q, pool, table, tl) for q in qs]
    outs = [torch.zeros_like(q) for q in qs]
    side = torch.cuda.Stream()
    graphs = []
    for q, o in zip(qs[:2], outs[:2]):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            for _ in range(4):
                qd.kv4_attention(q, pool, table, tl, out=o)
        graphs.append(gr)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        with torch.cuda.stream(streams[2]):
            qd.kv4_attention(qs[2], pool, table, tl, out=outs[2])
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_plan_append_attend_together():
    """A batch of uneven requests grown step by step from a captured graph: plan
    (in place), append, attend; compared with fp64 attention over all rows."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(12)
    nq, nkv, hd, page, B, W = 6, 2, 64, 16, 5, 8
    pages = 40
    pool = qd.kv4_pool(pages, nkv, hd, page, dev)
    table = torch.full((B, W), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    used, lens = _i64([0], dev), _i64([0] * B, dev)
    rows_new = [20, 1, 0, 33, 16]
    joins = _i64(rows_new, dev)
    # prompts
    n = sum(rows_new) + 2
    q = torch.randn(n, nq, hd, generator=g, device=dev)
    k, v = (torch.randn(n, nkv, hd, generator=g, device=dev) for _ in range(2))
    p = qd.kv4_plan(lens, joins, table, free, used, page, n, lens_out=lens, used_out=used)
    qd.kv4_append(k, v, pool, p.slots)
    _check_attention(q, pool, table, rows_new, p.cu_rows.tolist(), max_rows=33)
    # steps of one row each, from a graph
    joins = _i64([1] * B, dev)
    q, k, v = (torch.empty(B, h, hd, device=dev) for h in (nq, nkv, nkv))
    out = torch.zeros_like(q)

    def step():
        p = qd.kv4_plan(lens, joins, table, free, used, page, B, lens_out=lens, used_out=used)
        qd.kv4_append(k, v, pool, p.slots)
        qd.kv4_attention(q, pool, table, lens, cu_rows=p.cu_rows, out=out)

    keep = [x.clone() for x in (lens, used, table, pool)]
    step()
    for x, y in zip((lens, used, table, pool), keep):
        x.copy_(y)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        step()
    held = list(rows_new)
    for _ in range(20):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=dev))
        gr.replay()
        held = [h + 1 for h in held]
        assert lens.tolist() == held
        ref, size = P.attention(q, pool, table, held, list(range(B + 1)), hd ** -0.5, out)
        assert (out.double() - ref).abs().max() < 1e-4
    assert used.item() == sum(-(-h // page) for h in held)


def test_one_workspace_for_calls_of_different_shapes():
    """A workspace large enough for all serves any of them in turn: what one
    variant leaves in it does not reach the next."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(23)
    shapes = [(2, 1, 64, 1), (16, 2, 128, 1), (8, 1, 64, 4), (8, 1, 128, 4), (4, 1, 128, 1)]
    big = max(qd.kv4_attention_workspace(dev, nq, nkv, hd, rows).numel() for nq, nkv, hd, rows in shapes)
    ws = torch.zeros(big, dtype=torch.uint8, device=dev)
    made = []
    for nq, nkv, hd, rows in shapes:
        lens = [1500, 300, 77]
        pool, table = _context(lens, nkv, hd, 16, g, dev)
        cu = [0, rows, 2 * rows, 3 * rows]
        made.append((torch.randn(3 * rows, nq, hd, generator=g, device=dev), pool, table, lens, cu, rows))
    for _ in range(3):
        for q, pool, table, lens, cu, rows in made:
            _check_attention(q, pool, table, lens, cu, max_rows=rows, workspace=ws)


def test_refusals_on_the_gpu():
    """What the direct calls decline, the Python checks refuse by name; nothing is
    written."""
    qd, dev = _dev()
    pool = qd.kv4_pool(4, 2, 64, 16, dev)
    before = pool.clone()
    f = torch.randn(3, 2, 64, device=dev)
    i = _i64([0, 1, 2], dev)
    table = torch.zeros(3, 2, dtype=torch.int32, device=dev)
    free = torch.arange(4, dtype=torch.int32, device=dev)
    one = _i64([1], dev)
    q = torch.randn(3, 4, 64, device=dev)
    bad = [
        (TypeError, "int64", lambda: qd.kv4_append(f, f, pool, i.int())),
        (ValueError, "one element per row", lambda: qd.kv4_append(f, f, pool, i[:2])),
        (ValueError, "same shape", lambda: qd.kv4_append(f, f[:2], pool, i)),
        (ValueError, "same shape and dtype", lambda: qd.kv4_append(f, f.half(), pool, i)),
        (TypeError, "float32, bfloat16", lambda: qd.kv4_append(f.double(), f.double(), pool, i)),
        (ValueError, "kv heads", lambda: qd.kv4_append(f[:, :1], f[:, :1], pool, i)),
        (ValueError, "along head_dim", lambda: qd.kv4_append(f.transpose(0, 2), f.transpose(0, 2), pool, i)),
        (ValueError, "head_dim", lambda: qd.kv4_gather(pool, i, 32)),
        (ValueError, "no pages", lambda: qd.kv4_gather(pool, i, 128)),
        (ValueError, "contiguous", lambda: qd.kv4_gather(pool[:, :1], i, 64)),
        (ValueError, "CUDA", lambda: qd.kv4_gather(pool, i.cpu(), 64)),
        (ValueError, "multiple", lambda: qd.kv4_attention(q[:, :3], pool, table, i)),
        (ValueError, "per table row", lambda: qd.kv4_attention(q, pool, table, i[:2])),
        (ValueError, "cu_rows must have", lambda: qd.kv4_attention(q, pool, table, i, cu_rows=i)),
        (ValueError, "max_rows", lambda: qd.kv4_attention(q, pool, table, i, max_rows=0)),
        (ValueError, "max_rows", lambda: qd.kv4_attention(q, pool, table, i, max_rows=2)),
        (ValueError, "shape and dtype", lambda: qd.kv4_attention(q, pool, table, i, out=q[:2])),
        (ValueError, "overlap", lambda: qd.kv4_attention(q, pool, table, i, out=q[:1].expand(3, 4, 64))),
        (ValueError, "workspace", lambda: qd.kv4_attention(
            q, pool, table, i, workspace=torch.zeros(256, dtype=torch.uint8, device=dev))),
        (ValueError, "per table row", lambda: qd.kv4_plan(i[:2], i, table, free, one, 16, 4)),
        (ValueError, "page size", lambda: qd.kv4_plan(i, i, table, free, one, 17, 4)),
        (ValueError, "one element", lambda: qd.kv4_plan(i, i, table, free, i, 16, 4)),
        (ValueError, "negative", lambda: qd.kv4_plan(i, i, table, free, one, 16, -1)),
        (TypeError, "int32", lambda: qd.kv4_plan(i, i, table, free.long(), one, 16, 4)),
    ]
    for kind, msg, call in bad:
        with pytest.raises(kind, match=msg):
            call()
    assert torch.equal(pool, before) and not table.any()


def test_calls_on_another_stream_and_with_default_arguments():
    """The direct calls give what the checked ones give, on side streams too."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(31)
    lens = [100, 7]
    pool, table = _context(lens, 2, 64, 16, g, dev)
    q = torch.randn(2, 6, 64, generator=g, device=dev)
    tl = _i64(lens, dev)
    want = qd.kv4_attention(q, pool, table, tl, scale=64 ** -0.5)
    fast, qd._fast = qd._fast, None
    try:
        checked = qd.kv4_attention(q, pool, table, tl)
    finally:
        qd._fast = fast
    assert torch.equal(want, checked) and torch.equal(want, qd.kv4_attention(q, pool, table, tl))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [qd.kv4_attention(q, pool, table, tl) for _ in range(3)]
        k, v = qd.kv4_gather(pool, _i64([0, 5], dev), 64)
        other = torch.zeros_like(pool)
        qd.kv4_append(k, v, other, _i64([3, 4], dev))
    side.synchronize()
    for t in got:
        assert torch.equal(t, want)


@pytest.mark.parametrize("hd,nq,nkv,rows,t", [(128, 8, 2, 200, 30000), (64, 4, 2, 64, 60000), (128, 4, 1, 1, 50000)])
def test_long_contexts_do_not_drift(hd, nq, nkv, rows, t):
    """The MMAs truncate their accumulators; results over long contexts of fp32 rows
    stay within a few fp32 roundings all the same (the 2-norm over all rows: 4e-6,
    where fp32 sums over 60000 positions alone leave 2e-6 and accumulation in one
    MMA chain 4e-4)."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(t)
    pages = -(-t // 64)
    pool = torch.randint(0, 256, (pages, nkv, 64 * (hd + 8)), generator=g, device=dev, dtype=torch.uint8)
    par = torch.empty(pages, nkv, 2, 64, 2, device=dev)
    par[..., 0] = 0.2 + 0.2 * torch.rand(pages, nkv, 2, 64, generator=g, device=dev)
    par[..., 1] = -7.5 * par[..., 0]
    pool[..., 64 * hd:] = par.to(torch.bfloat16).view(torch.uint8).flatten(2)
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    q = torch.randn(rows, nq, hd, generator=g, device=dev)
    got = qd.kv4_attention(q, pool, table, _i64([t], dev), cu_rows=_i64([0, rows], dev), max_rows=rows)
    k, v = (x.transpose(0, 1).flatten(1, 2)[:, :t] for x in P.load(pool, hd))
    hide = torch.arange(t, device=dev) > t - rows + torch.arange(rows, device=dev)[:, None]
    ref = torch.empty(rows, nq, hd, dtype=torch.float64, device=dev)
    for h in range(nq):
        s = (q[:, h].double() * hd ** -0.5) @ k[h // (nq // nkv)].T
        ref[:, h] = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ v[h // (nq // nkv)]
    assert ((got.double() - ref).norm() / ref.norm()).item() < 4e-6
    # enough rows behind the request's for the kernel of many tiles
    q = torch.cat([q, q.new_zeros(-(-80 // nkv) * 128 * nkv // nq, nq, hd)])
    got = qd.kv4_attention(q, pool, table, _i64([t], dev), cu_rows=_i64([0, rows], dev), max_rows=rows)[:rows]
    assert ((got.double() - ref).norm() / ref.norm()).item() < 4e-6


@pytest.mark.parametrize("what", ["lens", "used"])
def test_large_plan_with_one_output_in_place(what):
    """A plan of many CTAs of which only the lengths, or only the cursor, are updated in place."""
    qd, dev = _dev()
    rng = random.Random(5)
    B, page = 900, 16
    lens = [rng.randrange(700) for _ in range(B)]
    joins = [rng.randrange(40) for _ in range(B)]
    table = [[rng.randrange(9999) for _ in range(64)] for _ in range(B)]
    free, used, rows = rng.sample(range(9999), 2000), 7, sum(joins) + 3000
    tl, tj, tu = _i64(lens, dev), _i64(joins, dev), _i64([used], dev)
    tt = torch.tensor(table, dtype=torch.int32, device=dev)
    p = qd.kv4_plan(tl, tj, tt, torch.tensor(free, dtype=torch.int32, device=dev), tu, page, rows,
                    lens_out=tl if what == "lens" else None, used_out=tu if what == "used" else None)
    got = dict(cu_rows=p.cu_rows.tolist(), lens=p.lens.tolist(), used=p.used.tolist(),
               slots=p.slots.tolist(), positions=p.positions.tolist(), table=tt.tolist())
    assert got == P.plan(lens, joins, table, free, used, page, rows)
    assert (tl.tolist() == lens) == (what == "used") and (tu.item() == used) == (what == "lens")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["slices", "odd", "heads"])
def test_strided_rows_of_many_tiles(dtype, layout):
    """Strided and unaligned rows, and out on top of q, where the tiles fill the GPU."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(31)
    rows, t = 1300, 1400
    pool, table = _context([t], 2, 64, 16, g, dev)
    q, out = _rows(rows, 8, 64, DTYPES[dtype], g, dev, layout)
    kw = dict(cu_rows=_i64([0, rows], dev), max_rows=rows)
    want = qd.kv4_attention(q.contiguous(), pool, table, _i64([t], dev), **kw)
    ref, size = P.attention(q, pool, table, [t], [0, rows], 64 ** -0.5, want, rows)
    assert (want.double() - ref).abs().max() < 0.02
    got = qd.kv4_attention(q, pool, table, _i64([t], dev), out=out, **kw)
    assert got is out and torch.equal(got, want)
    assert torch.equal(qd.kv4_attention(q, pool, table, _i64([t], dev), out=q, **kw), want)
    qd.check_status()


def test_few_tiles_and_many_tiles_agree():
    """The same request with and without rows behind it: two kernels, one result."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(32)
    pool, table = _context([700], 3, 128, 32, g, dev)
    q = torch.randn(3000, 9, 128, generator=g, device=dev)
    a = qd.kv4_attention(q[:300], pool, table, _i64([700], dev), cu_rows=_i64([0, 300], dev), max_rows=300)
    b = torch.full_like(q, 7.0)
    qd.kv4_attention(q, pool, table, _i64([700], dev), cu_rows=_i64([0, 300], dev), max_rows=300, out=b)
    assert (a - b[:300]).abs().max() < 2e-5 and (b[300:] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_any_scale(dtype, scale):
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(33)
    lens = [200, 0, 90]
    pool, table = _context(lens, 2, 128, 16, g, dev)
    q = torch.randn(200, 4, 128, generator=g, device=dev).to(DTYPES[dtype])
    _check_attention(q[:3], pool, table, lens, None, scale=scale)
    _check_attention(q, pool, table, lens, [0, 120, 120, 200], scale=scale, max_rows=120)


def test_lengths_below_zero_and_beyond_any_table():
    """Lengths that no caller should hold: nothing is seen, or all that the table has."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(34)
    pool, table = _context([64, 64, 64], 2, 64, 16, g, dev)
    for n, pad in ((1, 0), (70, 0), (70, 6000)):
        q = torch.randn(3 * n + pad, 4, 64, generator=g, device=dev)
        cu = _i64([0, n, 2 * n, 3 * n], dev)
        out = qd.kv4_attention(q, pool, table, _i64([-(1 << 62), -1, 1 << 62], dev), cu_rows=cu, max_rows=n)
        assert (out[:2 * n] == 0).all()
        full = qd.kv4_attention(q[2 * n:3 * n], pool, table[2:].repeat(n, 1)[:n], _i64([64] * n, dev))
        assert (out[2 * n:3 * n] - full).abs().max() < 2e-5
    qd.check_status()


def test_the_most_requests():
    """4096 requests in one call, some with prompts, against calls of 256 requests each."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(35)
    rng = random.Random(35)
    B, page, nkv, hd = 4096, 16, 2, 64
    rows = [rng.choice([0, 1, 1, 2]) if b % 97 else 90 for b in range(B)]
    lens = [max(n, rng.randrange(150)) for n in rows]
    W = 10
    table = torch.arange(B * W, dtype=torch.int32, device=dev).view(B, W)
    pool = torch.randint(0, 256, (B * W, nkv, page * (hd + 8)), generator=g, device=dev, dtype=torch.uint8)
    par = torch.rand(B * W, nkv, 2, page, 2, generator=g, device=dev)
    pool[..., page * hd:] = (par - torch.tensor([0.0, 1.5], device=dev)).to(torch.bfloat16).view(torch.uint8).flatten(2)
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + 5, 4, hd, generator=g, device=dev)
    out = torch.full_like(q, 0.25)
    qd.kv4_attention(q, pool, table, _i64(lens, dev), cu_rows=_i64(cu, dev), max_rows=90, out=out)
    assert (out[cu[-1]:] == 0.25).all()
    for b in range(0, B, 256):
        c = cu[b:b + 257]
        part = qd.kv4_attention(q[c[0]:c[-1]], pool, table[b:b + 256], _i64(lens[b:b + 256], dev),
                                cu_rows=_i64([x - c[0] for x in c], dev), max_rows=90)
        assert (part - out[c[0]:c[-1]]).abs().max() < 1e-4
    with pytest.raises(ValueError, match="4096"):
        qd.kv4_attention(q, pool, table[:1].repeat(4097, 1), torch.zeros(4097, dtype=torch.int64, device=dev),
                         cu_rows=torch.zeros(4098, dtype=torch.int64, device=dev), max_rows=90)
    qd.check_status()


def test_a_plan_in_a_graph_advances_the_state():
    """A captured plan, append and attention whose lengths and cursor are updated in place:
    every replay is the next step."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(36)
    B, page, nkv, hd, W = 5, 16, 2, 64, 8
    lens, used = _i64([0, 15, 16, 3, 40], dev), _i64([0], dev)
    start = lens.tolist()
    free = torch.arange(60, dtype=torch.int32, device=dev)
    table = torch.full((B, W), -1, dtype=torch.int32, device=dev)
    pool = P.empty_pool(60, nkv, hd, page, 0, dev)
    first = qd.kv4_plan(torch.zeros_like(lens), lens, table, free, used, page, sum(start), used_out=used)
    held = torch.randn(sum(start), nkv, hd, generator=g, device=dev)
    qd.kv4_append(held, -held, pool, first.slots)
    one, k = torch.ones_like(lens), torch.randn(B, nkv, hd, generator=g, device=dev)
    q, out = torch.randn(B, 4, hd, generator=g, device=dev), torch.zeros(B, 4, hd, device=dev)
    ws = qd.kv4_attention_workspace(dev, 4, nkv, hd)

    def step():
        plan = qd.kv4_plan(lens, one, table, free, used, page, B, lens_out=lens, used_out=used)
        qd.kv4_append(k, -k, pool, plan.slots)
        qd.kv4_attention(q, pool, table, plan.lens, out=out, workspace=ws)

    kept = [t.clone() for t in (lens, used, table)]
    step()
    for t, o in zip((lens, used, table), kept):
        t.copy_(o)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        step()
    for i in range(1, 30):
        k.normal_(generator=g)
        gr.replay()
        now = [n + i for n in start]
        assert lens.tolist() == now
        assert used.item() == sum(-(-n // page) for n in now)
        ref, _ = P.attention(q, pool, table, now, list(range(B + 1)), hd ** -0.5, out, 1)
        assert (out - ref).abs().max() < 1e-4
        own = [p for b, n in enumerate(now) for p in table[b, :-(-n // page)].tolist()]
        assert len(set(own)) == len(own) and min(own) >= 0
