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
