"""kv4_attention: calls that leave out arguments, and rows that nothing computes."""

import pytest

from tests import _kv4 as P

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _i64(x, dev):
    return torch.tensor(x, dtype=torch.int64, device=dev)


def _setup(rows, nq=4, t=60, B=3):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(51)
    pool = P.empty_pool(B * 4, 2, 64, 16, 0, dev)
    k, v = (torch.randn(B * 64, 2, 64, generator=g, device=dev) for _ in range(2))
    P.store(pool, 64, torch.arange(B * 64, device=dev), k, v)
    table = torch.arange(B * 4, dtype=torch.int32, device=dev).view(B, 4)
    return dev, pool, table, _i64([t] * B, dev), torch.randn(rows, nq, 64, generator=g, device=dev)


def _poison():
    """Leaves NaN in the memory that the next small tensors are made of."""
    for n in (1 << 10, 1 << 12, 1 << 14, 1 << 16, 1 << 20):
        for _ in range(4):
            torch.full((n,), float("nan"), device="cuda")


@pytest.mark.parametrize("checked", [False, True])
def test_rows_that_are_not_computed_are_zeros(checked, monkeypatch):
    """An output that the call makes has zeros where no request has a row, or one has more
    rows than max_rows."""
    from quartz_b200 import device as qd
    dev, pool, table, lens, q = _setup(12)
    if checked:
        monkeypatch.setattr(qd, "_fast", None)
    cu = _i64([0, 4, 5, 8], dev)
    want = torch.full_like(q, 7.0)
    qd.kv4_attention(q, pool, table, lens, cu_rows=cu, max_rows=4, out=want)
    assert (want[8:] == 7.0).all() and not (want[:8] == 7.0).any()
    for _ in range(3):
        _poison()
        got = qd.kv4_attention(q, pool, table, lens, cu_rows=cu, max_rows=4)
        assert torch.equal(got[:8], want[:8]) and (got[8:] == 0).all()
        _poison()
        got = qd.kv4_attention(q, pool, table, lens, cu_rows=cu, max_rows=1)
        assert (got[:4] == 0).all() and (got[5:] == 0).all() and (got[4] != 0).all()
        _poison()
        got = qd.kv4_attention(q, pool, table, lens)              # one row per request, nine more
        assert (got[3:] == 0).all() and (got[:3] != 0).all()
        _poison()
        assert (qd.kv4_attention(q, pool, table[:0], lens[:0]) == 0).all()
        assert torch.equal(qd.kv4_attention(q[:2], pool, table, lens), got[:2])
    qd.check_status()


@pytest.mark.parametrize("checked", [False, True])
def test_max_rows_left_out_takes_all_rows(checked, monkeypatch):
    from quartz_b200 import device as qd
    dev, pool, table, lens, q = _setup(50)
    if checked:
        monkeypatch.setattr(qd, "_fast", None)
    for rows in ([4, 0, 1], [46, 3, 1], [50, 0, 0], [0, 0, 0]):
        cu = _i64([0, rows[0], rows[0] + rows[1], sum(rows)], dev)
        want = qd.kv4_attention(q, pool, table, lens, cu_rows=cu, max_rows=50)
        assert torch.equal(qd.kv4_attention(q, pool, table, lens, cu_rows=cu), want)
        assert torch.equal(qd.kv4_attention(q, pool, table, lens, cu_rows=cu, max_rows=None), want)
        ref, _ = P.attention(q, pool, table, [60] * 3, cu.tolist(), 64 ** -0.5, torch.zeros_like(q))
        assert (want - ref).abs().max() < 1e-4
    # no rows at all
    assert qd.kv4_attention(q[:0], pool, table, lens, cu_rows=_i64([0] * 4, dev)).shape == (0, 4, 64)
    qd.check_status()


def test_a_cuda_failure_is_raised_and_not_tried_again(monkeypatch):
    """A launch may be queued when the library reports a CUDA error (attention has two):
    the direct calls raise it, and the checked ones do not run after them."""
    import ctypes

    from quartz_b200 import _lib, device as qd
    dev, pool, table, lens, q = _setup(3)
    want = qd.kv4_attention(q, pool, table, lens)
    if qd._fast is None:
        pytest.skip("the _fastcall extension is not built")
    lib, calls = _lib.load(), []
    names = ("qz_kv4_plan", "qz_kv4_append", "qz_kv4_gather", "qz_kv4_attention",
             "qz_kv4_attention_workspace_bytes", "qz_last_error")
    real = [ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names]

    def fails(kind):
        sig, res = _lib.SIGNATURES[kind]
        return ctypes.CFUNCTYPE(res, *sig)(lambda *a: calls.append(kind) or 2)     # QZ_ERR_CUDA

    fakes = [fails(n) for n in names[:4]]
    one = torch.ones(3, dtype=torch.int64, device=dev)
    free = torch.arange(4, dtype=torch.int32, device=dev)
    k = q[:, :2].contiguous()
    lib.qz_kv4_gather(None, 0, 0, 0, 0, None, 0, None, None, None)      # leaves a message
    try:
        qd._fast.bind(_lib.QuartzError, *(ctypes.cast(f, ctypes.c_void_p).value for f in fakes), *real[4:])
        for name in names[:4]:                                         # the library, called past the fakes
            monkeypatch.setattr(lib, name, lambda *a: pytest.fail("tried again"))
        for call in (lambda: qd.kv4_plan(lens, one, table, free, one[:1], 16, 4),
                     lambda: qd.kv4_append(k, k, pool, lens),
                     lambda: qd.kv4_gather(pool, lens, 64),
                     lambda: qd.kv4_attention(q, pool, table, lens)):
            with pytest.raises(_lib.QuartzError, match="n_kv"):
                call()
    finally:
        qd._fast.bind(_lib.QuartzError, *real)
    assert calls == list(names[:4])
    monkeypatch.undo()
    assert torch.equal(qd.kv4_attention(q, pool, table, lens), want)
