"""How close kv4_attention comes to 64 bits, at the places where a form with fewer
bits would show: the rounding of 16-bit rows, V rows of very different size, long
contexts."""

import math

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


def _pool_of(k, v, page):
    """A pool of one request's rows k, v [t, n_kv, hd] in order, and its table."""
    t, nkv, hd = k.shape
    pages = -(-t // page)
    pool = P.empty_pool(pages, nkv, hd, page, 0, k.device)
    P.store(pool, hd, torch.arange(t, device=k.device), k, v)
    return pool, torch.arange(pages, dtype=torch.int32, device=k.device)[None]


def _exact(q, pool, t, rows):
    """fp64 result of the last `rows` positions' queries q [rows, nq, hd], and per
    element sum_t p_t |v_t|."""
    hd, nq, nkv = q.shape[2], q.shape[1], pool.shape[1]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    size = torch.empty_like(out)
    hide = torch.arange(t, device=q.device) > t - rows + torch.arange(rows, device=q.device)[:, None]
    for h in range(nkv):
        k, v = (x.transpose(0, 1).flatten(1, 2)[0, :t] for x in P.load(pool[:, h:h + 1], hd))
        for j in range(h * (nq // nkv), (h + 1) * (nq // nkv)):
            s = (q[:, j].double() * hd ** -0.5) @ k.T
            p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
            out[:, j], size[:, j] = p @ v, p @ v.abs()
    return out, size


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype,most", [("fp16", 0.04), ("bf16", 0.005)])
def test_prompts_of_16_bits_round_once(dtype, most, hd):
    """The tiles' results in 16 bits are the exact ones rounded once, but where those
    lie next to a border between two values. An error e before the rounding crosses a
    border for a share |e| / ulp of the results, and an ulp is 2^-11 to 2^-10 of a
    fp16 value, 2^-8 to 2^-7 of a bf16 one. Scores that are off by an eighth of the
    worst case 4 A (hd / 16 + 8) 2^-23, A = 8, give 8e-6 and 1.2 % or 0.15 % of the
    results; a weight in one fp16 limb gives 2^-12 / sqrt(3) of it, 16 % or 2 %."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(41)
    rows, t, nkv, nq = 1300, 1400, 2, 8              # 82 tiles: the tensor cores' kernel
    k, v = (torch.randn(t, nkv, hd, generator=g, device=dev) for _ in range(2))
    pool, table = _pool_of(k, v, 32)
    q = torch.randn(rows, nq, hd, generator=g, device=dev).to(DTYPES[dtype])
    got = qd.kv4_attention(q, pool, table, _i64([t], dev), cu_rows=_i64([0, rows], dev), max_rows=rows)
    ref, _ = _exact(q, pool, t, rows)
    other = (got != ref.to(got.dtype)).double().mean().item()
    assert other < most, other
    qd.check_status()


# rows of the request, heads: one row and a few take the split kernel with one and two
# blocks of queries, 1300 rows the tiles
FORMS = {"one": (1, 8), "few": (5, 8), "tiles": (1300, 8)}


def _check_sums(got, ref, size, score_err):
    """|got - ref| <= size (2 score_err + 2^-19) and the rounding: every weight is off by
    the error of its score and 2^-20 of exponent and split, the sum of the weights too,
    and size is the sum of the weighted |v|."""
    eps = torch.finfo(got.dtype).eps / 2
    bound = size * (2 * score_err + 2.0 ** -19) + ref.abs() * eps + torch.finfo(got.dtype).tiny
    assert torch.isfinite(got).all()
    over = ((got.double() - ref).abs() / bound).max().item()
    assert over <= 1, over


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("at", [(0, 77), (900, 1350), (100, 2300, 4000)])
@pytest.mark.parametrize("ratio", [12, 24, 40, 100])
def test_a_large_value_without_weight_costs_nothing(ratio, at, form, hd, dtype):
    """Some V rows 2^ratio times the others, with 2^-100 of the weight and less: their p |v|
    is nothing, and the result is what fp32 sums of p v give. The ordinary scores have
    A = scale * sum |q k| below 20 (128 products of unit normals, and 8 * 0.3), so they
    are off by at most 4 A (hd / 16 + 8) 2^-23; those rows' A is larger, but not their
    share."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(ratio)
    rows, nq = FORMS[form]
    nkv, t = 2, 1400 if max(at) < 1400 else 4200
    k, v = (torch.randn(t, nkv, hd, generator=g, device=dev) for _ in range(2))
    q = torch.randn(rows, nq, hd, generator=g, device=dev).to(DTYPES[dtype])
    # along dimension 0 the queries have 8 and only those keys anything: their scores lie
    # scale * 8 * x = 70 + ratio ln 2 below the others', about
    q[..., 0], k[..., 0] = 8.0, 0.0
    for p in at:
        k[p] = 0.0
        k[p, :, 0] = -(70 + ratio * math.log(2)) / 8 * hd ** 0.5
        v[p] *= 2.0 ** ratio
    pool, table = _pool_of(k, v, 16)
    got = qd.kv4_attention(q, pool, table, _i64([t], dev), cu_rows=_i64([0, rows], dev), max_rows=rows)
    ref, size = _exact(q, pool, t, rows)
    _check_sums(got, ref, size, 4 * 20 * (hd / 16 + 8) * 2.0 ** -23)
    qd.check_status()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["zero", "constant", "tiny"])
def test_a_position_that_takes_the_weight_but_has_no_value(kind, form, dtype):
    """The first position has nearly all the weight and a V row of zeros (or of one value,
    with no steps, or of 2^-40): what the others add is small and still theirs."""
    qd, dev = _dev()
    hd, nkv, t = 64, 2, 1400
    g = torch.Generator(device=dev).manual_seed(7)
    rows, nq = FORMS[form]
    k, v = (torch.randn(t, nkv, hd, generator=g, device=dev) for _ in range(2))
    q = torch.randn(rows, nq, hd, generator=g, device=dev).to(DTYPES[dtype])
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[0] = 0.0
    k[0, :, 0] = 40.0                                   # a score of 40, e^40 = 2^58
    v[0] = {"zero": 0.0, "constant": 2.0 ** -30, "tiny": 2.0 ** -40}[kind] * (v[0] if kind == "tiny" else 1)
    pool, table = _pool_of(k, v, 16)
    got = qd.kv4_attention(q, pool, table, _i64([t], dev), cu_rows=_i64([0, rows], dev), max_rows=rows)
    ref, size = _exact(q, pool, t, rows)
    # the first position's score has A = 40, and all weights are relative to it
    _check_sums(got, ref, size, 4 * 40 * (hd / 16 + 8) * 2.0 ** -23)
    qd.check_status()


@pytest.mark.parametrize("dtype,most", [("fp16", 0.28), ("bf16", 0.035)])
@pytest.mark.parametrize("hd,B,rows", [(64, 93, 1), (64, 40, 5), (128, 74, 1)])
def test_long_contexts_of_16_bits_do_not_drift(hd, B, rows, dtype, most):
    """So many requests that a CTA takes whole contexts of 2^19 positions: results are the
    exact ones rounded once, but for a share |e| / ulp (see
    test_prompts_of_16_bits_round_once). Here the results are small differences of the
    sums: with steps of 0.3 and zeros of -7.5 steps, sum p s (c - 8) and sum p (z + 8 s)
    are -0.15 and 0.15 of sum p, and the results, 1.4 times the root of
    exp(1.4^2) / 2^19, are 5e-3 of it. A chain of 128 truncating MMAs is 128 * 3e-8 / 2 =
    2e-6 of 0.15 low, and fp32 sums of 2^14 terms a lane are off by up to
    128 * 2^-25 = 4e-6 of it: 9e-7 together. An ulp is 5e-3 * 2^-10.5 = 3.5e-6 (fp16) or
    2.8e-5 (bf16): shares of 26 % and 3.2 %, with the scores' 1.2 % and 0.15 %. One chain
    over a warp's 2^17 positions is 2^14 * 3e-8 / 2 = 2.5e-4 of 0.15 low, more than an ulp
    of either."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(hd + B)
    nkv, nq, t, page = 8, 16, 1 << 19, 256
    if torch.cuda.mem_get_info(0)[0] < 8 << 30:
        pytest.skip("needs 8 GB of device memory")
    pages = t // page
    pool = torch.randint(0, 256, (pages, nkv, page * (hd + 8)), generator=g, device=dev, dtype=torch.uint8)
    par = torch.empty(pages, nkv, 2, page, 2, device=dev)
    par[..., 0] = 0.2 + 0.2 * torch.rand(pages, nkv, 2, page, generator=g, device=dev)
    par[..., 1] = -7.5 * par[..., 0]
    pool[..., page * hd:] = par.to(torch.bfloat16).view(torch.uint8).flatten(2)
    table = torch.arange(pages, dtype=torch.int32, device=dev).expand(B, pages).contiguous()
    q = torch.randn(B * rows, nq, hd, generator=g, device=dev).to(DTYPES[dtype])
    lens = _i64([t] * B, dev)
    cu = _i64([b * rows for b in range(B + 1)], dev)
    got = qd.kv4_attention(q, pool, table, lens, cu_rows=cu, max_rows=rows)
    other = []
    for b in (0, B // 2):
        at = slice(b * rows, (b + 1) * rows)
        ref, _ = _exact(q[at], pool, t, rows)
        other.append((got[at] != ref.to(got.dtype)).double().mean().item())
    assert max(other) < most, other
    qd.check_status()


def test_one_workspace_for_tiles_and_long_contexts():
    """A workspace that calls of both kernels, head sizes and types share in turn, with
    items longer than the places where sums are moved to it."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(24)
    shapes = [(8, 2, 128, 1300, 1500, "fp32"), (8, 2, 64, 1300, 4500, "bf16"), (16, 8, 64, 1, 40000, "fp16"),
              (8, 2, 64, 1300, 1400, "fp32"), (8, 2, 128, 1300, 4500, "fp16"), (4, 1, 128, 1, 40000, "bf16")]
    ws = torch.zeros(max(qd.kv4_attention_workspace(dev, nq, nkv, hd, rows).numel()
                         for nq, nkv, hd, rows, _, _ in shapes), dtype=torch.uint8, device=dev)
    made = []
    for nq, nkv, hd, rows, t, dtype in shapes:
        k, v = (torch.randn(t, nkv, hd, generator=g, device=dev) for _ in range(2))
        pool, table = _pool_of(k, v, 16)
        q = torch.randn(rows, nq, hd, generator=g, device=dev).to(DTYPES[dtype])
        args = (q, pool, table, _i64([t], dev))
        kw = dict(cu_rows=_i64([0, rows], dev), max_rows=rows)
        want = qd.kv4_attention(*args, **kw, workspace=qd.kv4_attention_workspace(dev, nq, nkv, hd, rows))
        _check_sums(want, *_exact(q, pool, t, rows), 4 * 20 * (hd / 16 + 8) * 2.0 ** -23)
        made.append((args, kw, want))
    for _ in range(3):
        for args, kw, want in made:
            assert torch.equal(qd.kv4_attention(*args, **kw, workspace=ws), want)
    qd.check_status()


def test_a_place_of_the_workspace_has_one_owner():
    """The tiles' fp32 sums go to places of the workspace (one for each SM, its last part)
    that a CTA takes and leaves: places marked as taken stay as they are, whatever SM a
    CTA runs on, and the others are free again afterwards."""
    qd, dev = _dev()
    g = torch.Generator(device=dev).manual_seed(25)
    rows, t, nkv, nq, hd = 1300, 4500, 2, 8, 64      # 82 tiles of 36 steps: sums every 16
    k, v = (torch.randn(t, nkv, hd, generator=g, device=dev) for _ in range(2))
    pool, table = _pool_of(k, v, 32)
    q = torch.randn(rows, nq, hd, generator=g, device=dev).to(torch.bfloat16)
    args, kw = (q, pool, table, _i64([t], dev)), dict(cu_rows=_i64([0, rows], dev), max_rows=rows)
    want = qd.kv4_attention(*args, **kw)
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    ws = qd.kv4_attention_workspace(dev, nq, nkv, hd, rows)
    taken = ws[20 * sms:24 * sms].view(torch.int32)  # behind five tickets an SM
    sums = ws[-sms * 128 * hd * 4:].view(sms, -1)
    held = torch.arange(sms, device=dev) % 3 == 0
    assert sms - held.sum() >= 82
    taken[held] = 1
    sums[held] = 0xAB
    for _ in range(3):
        assert torch.equal(qd.kv4_attention(*args, **kw, workspace=ws), want)
        assert torch.equal(taken, held.int()) and (sums[held] == 0xAB).all()
    assert (sums[~held] != 0).any()
    qd.check_status()


@pytest.mark.parametrize("seed", range(48))
def test_uneven_requests_of_any_scale(seed):
    """Requests of uneven rows and lengths with V rows of very different size, rows of zeros
    and offsets among them. Per row, an error is at most sum_t p_t max_d |v_td| times that of
    the weights: exp(2 e) - 1 for scores off by e = 4 A (hd / 16 + 8) 2^-23, A the row's
    largest scale * sum |q k|, and 2^-19 of exponent, split and sums; values of 2^90 times a
    row's own may take 2^-95 of themselves; then the rounding."""
    import random
    qd, dev = _dev()
    rng, g = random.Random(seed), torch.Generator(device=dev).manual_seed(seed)
    hd, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128, 256])
    nkv, group = rng.choice([(1, 16), (2, 4), (3, 5), (8, 2), (2, 1), (1, 3)])
    dtype = DTYPES[rng.choice(["fp32", "fp32", "bf16"])]
    rows = [rng.choice([0, 1, 2, 5, rng.randrange(1, 900)]) for _ in range(rng.choice([1, 2, 3, 7]))]
    lens = [max(0, n + rng.choice([-3, 0, 0, 1, rng.randrange(3000)])) for n in rows]
    spread, shift = rng.choice([0, 4, 12, 30, 60]), rng.choice([0, 1, 30])
    B, width = len(rows), max(1, -(-max(lens) // page))
    order = torch.randperm(B * width + 1, generator=g, device=dev).to(torch.int32)
    table = order[:B * width].view(B, width).contiguous()
    pool = P.empty_pool(B * width + 1, nkv, hd, page, 0xFF, dev)
    for b, t in enumerate(lens):
        if not t:
            continue
        k, v = (torch.randn(t, nkv, hd, generator=g, device=dev) for _ in range(2))
        e = (torch.randn(t, nkv, 1, generator=g, device=dev) * spread).clamp(-100, 100)
        v = (v + shift * torch.randn(t, nkv, 1, generator=g, device=dev)) * torch.exp2(e)
        v[torch.rand(t, generator=g, device=dev) < rng.choice([0, 0.1])] = 0
        pos = torch.arange(t, device=dev)
        P.store(pool, hd, table[b][pos // page].long() * page + pos % page, k * rng.choice([1, 3]), v)
    cu = [sum(rows[:b]) for b in range(B + 1)]
    q = torch.randn(cu[-1] + rng.choice([0, 3, 2000]) + 1, nkv * group, hd, generator=g, device=dev)
    q = (q * rng.choice([1, 4])).to(dtype)
    out = torch.full_like(q, 0.25)
    qd.kv4_attention(q, pool, table, _i64(lens, dev), cu_rows=_i64(cu, dev), max_rows=max(1, *rows), out=out)
    assert (out[cu[-1]:] == 0.25).all()
    keys, vals = P.load(pool, hd)
    for b, (n, t) in enumerate(zip(rows, lens)):
        pos = torch.arange(t, device=dev)
        at = table[b][pos // page].long(), pos % page
        hide = pos > t - n + torch.arange(n, device=dev)[:, None]
        for h in range(nkv * group if n and t else 0):
            k, v = keys[at[0], h // group, at[1]], vals[at[0], h // group, at[1]]
            x = q[cu[b]:cu[b + 1], h].double() * hd ** -0.5
            p = torch.nan_to_num(torch.softmax((x @ k.T).masked_fill(hide, -math.inf), -1), nan=0.0)
            score = 4 * (x.abs() @ k.abs().T).masked_fill(hide, 0).amax(-1, keepdim=True) * (hd / 16 + 8) * 2.0 ** -23
            ref, size = p @ v, p @ v.abs().amax(-1, keepdim=True)
            bound = size * ((2 * score).exp() - 1 + 2.0 ** -19) + v.abs().max() * 2.0 ** -95
            bound = bound + ref.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny
            got = out[cu[b]:cu[b + 1], h].double()
            assert ((got - ref).abs() <= bound).all(), (b, h, ((got - ref).abs() / bound).max().item())
        if n and not t:
            assert (out[cu[b]:cu[b + 1]] == 0).all()
    qd.check_status()
