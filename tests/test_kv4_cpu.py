"""Refusals of the paged 4-bit cache's entry points, without a GPU: the C ABI
checks its arguments before it touches the device, the Python calls before they
touch the library."""

import pytest

torch = pytest.importorskip("torch")

INVALID = 1
P16 = 1 << 12      # an aligned non-null "pointer" (never read: the call is refused first)


def _lib():
    from quartz_b200 import _lib
    return _lib


def _plan(**kw):
    a = dict(lens=P16, joins=P16, B=4, table=P16, width=8, free=P16, n_free=9, used=P16, page=16,
             rows=4, cu=P16, lens_out=P16, used_out=P16, slots=P16, pos=P16, stream=None)
    a.update(kw)
    return _lib().load().qz_kv4_plan(*a.values())


def _append(**kw):
    a = dict(k=P16, v=P16, dtype=0, krs=128, khs=64, vrs=128, vhs=64, n=4, nkv=2, hd=64, pool=P16,
             pages=9, page=16, slots=P16, stream=None)
    a.update(kw)
    return _lib().load().qz_kv4_append(*a.values())


def _rope(**kw):
    a = dict(qkv=P16, qn=None, kn=None, inv=P16, q_out=P16, M=4, nq=4, nkv=2, hd=64, pos=P16,
             pool=P16, pages=9, page=16, slots=P16, eps=1e-6, stream=None)
    a.update(kw)
    return _lib().load().qz_qk_rope_kv4(*a.values())


def _gather(**kw):
    a = dict(pool=P16, pages=9, page=16, nkv=2, hd=64, slots=P16, n=4, k=P16, v=P16, stream=None)
    a.update(kw)
    return _lib().load().qz_kv4_gather(*a.values())


def _attend(**kw):
    a = dict(q=P16, dtype=0, qrs=256, qhs=64, out=P16, ors=256, ohs=64, pool=P16, pages=9, page=16,
             table=P16, width=8, lens=P16, cu=None, B=3, n=3, max_rows=1, nq=4, nkv=2, hd=64,
             scale=1.0, ws=P16, ws_bytes=0, stream=None)
    a.update(kw)
    return _lib().load().qz_kv4_attention(*a.values())


@pytest.mark.parametrize("call,kw,msg", [
    (_plan, dict(B=0), "requests must be"), (_plan, dict(B=4097), "requests must be"),
    (_plan, dict(page=24), "page size"), (_plan, dict(page=512), "page size"),
    (_plan, dict(width=0), "table width"), (_plan, dict(width=1 << 27), "table width"),
    (_plan, dict(n_free=-1), "free-page"), (_plan, dict(rows=-1), "row count"),
    (_plan, dict(lens=None), "null pointer"), (_plan, dict(free=None), "null pointer"),
    (_plan, dict(slots=None), "null pointer"), (_plan, dict(used_out=None), "null pointer"),
    (_append, dict(hd=96), "head_dim"), (_append, dict(page=8), "page size"),
    (_append, dict(nkv=0), "n_kv"), (_append, dict(pages=0), "page count"),
    (_append, dict(pool=None), "pool"), (_append, dict(pool=P16 + 8), "pool"),
    (_append, dict(dtype=3), "dtype"), (_append, dict(n=-1), "row count"),
    (_append, dict(k=None), "null pointer"), (_append, dict(slots=None), "null pointer"),
    (_rope, dict(nq=3), "multiple"), (_rope, dict(hd=32), "head_dim"), (_rope, dict(M=-1), "row count"),
    (_rope, dict(qn=P16), "both norm weights"), (_rope, dict(pos=None), "null pointer"),
    (_rope, dict(page=0), "page size"),
    (_gather, dict(hd=256), "head_dim"), (_gather, dict(k=P16 + 4), "16-byte"),
    (_gather, dict(v=None), "null pointer"), (_gather, dict(n=-1), "row count"),
    (_attend, dict(nq=5), "multiple"), (_attend, dict(nq=0), "multiple"),
    (_attend, dict(hd=80), "head_dim"), (_attend, dict(page=17), "page size"),
    (_attend, dict(dtype=-1), "dtype"), (_attend, dict(B=4097), "requests must be"),
    (_attend, dict(n=-1), "row count"), (_attend, dict(width=0), "table width"),
    (_attend, dict(width=(1 << 26) + 1), "table width"),
    (_attend, dict(max_rows=0), "max_rows"), (_attend, dict(max_rows=2), "max_rows"),
    (_attend, dict(lens=None), "null pointer"), (_attend, dict(ws=None), "null pointer"),
])
def test_c_abi_refuses(call, kw, msg):
    assert call(**kw) == INVALID
    assert msg in _lib().last_error()


def test_nothing_to_do_is_no_error():
    assert _append(n=0, k=None, v=None, slots=None) == 0
    assert _gather(n=0, k=None, v=None, slots=None) == 0
    assert _attend(n=0, q=None, out=None) == 0
    assert _attend(B=0, table=None, lens=None) == 0


def test_python_calls_refuse_before_the_library():
    from quartz_b200 import device as qd
    f, i = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int64)
    pool = torch.zeros(3, 2, 16 * 72, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        qd.kv4_append(f, f, pool, i)
    with pytest.raises(ValueError, match="CUDA"):
        qd.kv4_gather(pool, i, 64)
    with pytest.raises(ValueError, match="CUDA"):
        qd.kv4_attention(f, pool, torch.zeros(2, 4, dtype=torch.int32), i)
    with pytest.raises(ValueError, match="CUDA"):
        qd.kv4_plan(i, i, torch.zeros(2, 4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32),
                    i[:1], 16, 4)
    with pytest.raises(TypeError):
        qd.kv4_append([1], [2], pool, i)
    with pytest.raises(ValueError, match="page_size"):
        qd.kv4_block_bytes(20, 64)
    with pytest.raises(ValueError, match="head_dim"):
        qd.kv4_block_bytes(16, 96)
    assert qd.kv4_block_bytes(16, 128) == 16 * 136


def test_the_oracle_reads_back_what_it_stored():
    """The tests' own statement of the layout is consistent: store then load."""
    from tests import _kv4 as P
    g = torch.Generator().manual_seed(0)
    for hd, page in ((64, 16), (128, 32)):
        pool = P.empty_pool(4, 2, hd, page)
        k, v = (torch.randn(9, 2, hd, generator=g) for _ in range(2))
        slots = torch.randperm(4 * page, generator=g)[:9]
        P.store(pool, hd, slots, k, v)
        gk, gv = P.load(pool, hd)
        assert torch.equal(gk[slots // page, :, slots % page], P.values(k))
        assert torch.equal(gv[slots // page, :, slots % page], P.values(v))
        # within half a step of the row (and |z| 2^-9 at its lower end)
        span = (k.amax(-1) - k.amin(-1)).double()
        err = (P.values(k) - k.double()).abs().amax(-1)
        assert (err <= span / 30 * (1 + 2.0 ** -7) + k.abs().amax(-1) * 2.0 ** -8).all()
