"""Device-level entry points over torch CUDA tensors (no host copies).

Each function validates its tensors, then calls the C ABI on the current torch
stream. Outputs may be passed in (written in place, like the reference's
out-parameters) or are allocated here. torch is used only for device memory
and streams.

    gemv(q, scale, x)            -> y        quartz/kernels/int8.py:24-38
    gemm(q, scale, X)            -> Y        quartz/kernels/int8.py:66-87
    fused_mlp(gu_q, gu_s, x, down_q, down_s)  -> out   quartz/kernels/fused.py:27-65
    silu_mul(gu)                 -> a        quartz/quantize.py:112-114 (+ ops.py:35-37)

Decode-step glue (the fp32 work between the int8 matmuls of one token):

    embed_gather(q, scale, ids)  -> rows     quartz/quantize.py:78-80
    rmsnorm(x, w, eps)           -> y        quartz/ops.py:24-32
    qk_rope(qkv, ...)            -> q        quartz/models/qwen3.py:31-41, rope.py:47-78
    attention_decode(q, kc, vc, T)           quartz/attention.py:29-43 (one query row)
    attention_decode_qkv(qkv, ...)           the two above plus the KV append, one launch
    attention_prefill(q, kc, vc, pos0)       quartz/attention.py:15-43 (causal rows)
    argmax(logits)               -> tokens   quartz/sample.py:21-22

Paged 4-bit KV cache (no counterpart in quartz): sequences of uneven length
over one pool of pages. ``quartz_b200.paged`` decodes with it.

    kv4_pool(pages, n_kv, hd, page_size)       the zeroed pool of one layer
    kv4_plan(lens, new_rows, table, free, used, page_size, rows)
                                               block tables, slots, positions
    kv4_append(k, v, pool, slots)              quantise and store rows
    kv4_gather(pool, slots, hd)  -> k, v       the values the rows stand for
    qk_rope_kv4(qkv, ...)        -> q          q/k norm, RoPE and append in one launch
    kv4_attention(q, pool, table, lens, ...)   one row, a few rows or a prompt
"""

from __future__ import annotations

import ctypes
import threading
import warnings
from typing import NamedTuple

import torch

from . import _lib

_init_lock = threading.Lock()
_fast = None     # the extension module _fastcall, once a device is ready
_ready_devices: set[int] = set()
_mlp_ws: dict[int, torch.Tensor] = {}
_gemm_ws: dict[int, torch.Tensor] = {}


# The current stream's raw handle without building a torch.cuda.Stream object
# (a few microseconds of host time in every call).
_raw_stream_fn = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr(dev: torch.device) -> int:
    if _raw_stream_fn is not None and dev.index is not None:
        return _raw_stream_fn(dev.index)
    return torch.cuda.current_stream(dev).cuda_stream


def ensure_device(dev: torch.device | int | None = None) -> int:
    """qz_init once per device (checks that it is an sm_100 GPU)."""
    if _ready_devices:                      # the per-call path: no availability probe
        idx = dev.index if isinstance(dev, torch.device) else dev
        if idx is None:
            idx = torch.cuda.current_device()
        if idx in _ready_devices:
            return idx
    if not torch.cuda.is_available():
        raise RuntimeError("quartz_b200 needs a CUDA device; none is available")
    if dev is None:
        idx = torch.cuda.current_device()
    elif isinstance(dev, int):
        idx = dev
    else:
        idx = dev.index if dev.index is not None else torch.cuda.current_device()
    if idx not in _ready_devices:
        with _init_lock:
            if idx not in _ready_devices:
                with torch.cuda.device(idx):
                    _lib.check(_lib.load().qz_init(idx))
                _bind_fast(idx)
                _ready_devices.add(idx)
    return idx


def _bind_fast(idx: int) -> None:
    """Give _fastcall (csrc/fastcall.cpp) the library's entry points and a ready device."""
    global _fast
    if _fast is None:
        try:
            from . import build
            built, want = build.fast_stamp(), build.fast_tag()
            if built != want:
                raise ImportError(f"built for {built or 'nothing'}, this is {want}")
            from . import _fastcall
        except ImportError as e:      # the same kernels, 4 to 9 us more for each paged-cache call
            warnings.warn(f"quartz_b200/_fastcall.so does not load ({e}): build it with "
                          "`python -m quartz_b200.build`", RuntimeWarning, stacklevel=3)
            return
        lib = _lib.load()
        _fastcall.bind(_lib.QuartzError, *(
            ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in (
                "qz_kv4_plan", "qz_kv4_append", "qz_kv4_gather", "qz_kv4_attention",
                "qz_kv4_attention_workspace_bytes", "qz_last_error")))
        _fast = _fastcall
    _fast.device_ready(idx)


def _same_device(dev: torch.device, *ts) -> None:
    for t in ts:
        if t is not None and t.device != dev:
            raise ValueError(f"all tensors must be on {dev}, found one on {t.device}")


def _need(t: torch.Tensor, dtype, name: str, ndim: int | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D, got shape {tuple(t.shape)}")


def _weights(q, scale, name="q"):
    _need(q, torch.int8, name, 2)
    _need(scale, torch.float32, name + " scale", 2)
    N, K = q.shape
    if scale.shape[0] != N:
        raise ValueError(f"{name}: scale has {scale.shape[0]} rows, weights have {N}")
    ng = scale.shape[1]
    if ng < 1 or K % ng:
        raise ValueError(f"scale has {ng} groups that do not tile K={K}")
    return N, K, ng


def _ptr(t):
    return None if t is None else t.data_ptr()


def gemv(q, scale, x, y=None, residual=None, norm_w=None, eps=1e-6):
    """y[n] = sum_g scale[n,g] sum_{j<G} x[gG+j] q[n,gG+j] (+ residual[n]).
    With norm_w, the GEMV of RMSNorm(x) * norm_w (normalised in the kernel)."""
    N, K, ng = _weights(q, scale)
    ensure_device(q.device)
    _need(x, torch.float32, "x")
    if x.numel() != K:
        raise ValueError(f"x has {x.numel()} elements, expected K={K}")
    if y is None:
        y = torch.empty(N, dtype=torch.float32, device=q.device)
    _need(y, torch.float32, "y")
    if y.numel() != N:
        raise ValueError(f"y has {y.numel()} elements, expected N={N}")
    if residual is not None:
        _need(residual, torch.float32, "residual")
        if residual.numel() != N:
            raise ValueError("residual must have N elements")
    _same_device(q.device, scale, x, y, residual, norm_w)
    with torch.cuda.device(q.device):
        if norm_w is not None:
            _need(norm_w, torch.float32, "norm_w", 1)
            if norm_w.numel() != K:
                raise ValueError("norm_w must have K elements")
            scratch = torch.empty(K, dtype=torch.float32, device=q.device)
            _lib.check(_lib.load().qz_gemv_w8_rmsnorm(
                q.data_ptr(), scale.data_ptr(), ng, x.data_ptr(), norm_w.data_ptr(), float(eps),
                y.data_ptr(), N, K, _ptr(residual), scratch.data_ptr(), _stream_ptr(q.device)))
            return y
        _lib.check(_lib.load().qz_gemv_w8(q.data_ptr(), scale.data_ptr(), ng, x.data_ptr(),
                                          y.data_ptr(), N, K, _ptr(residual),
                                          _stream_ptr(q.device)))
    return y


def gemm(q, scale, X, Y=None, residual=None):
    """Y[m, n] for each row m of X [M, K] (+ residual[m, n])."""
    N, K, ng = _weights(q, scale)
    ensure_device(q.device)
    _need(X, torch.float32, "X")
    if X.dim() != 2 or X.shape[1] != K:
        raise ValueError(f"X must be [M, {K}], got {tuple(X.shape)}")
    M = X.shape[0]
    if Y is None:
        Y = torch.empty((M, N), dtype=torch.float32, device=q.device)
    _need(Y, torch.float32, "Y")
    if Y.numel() != M * N:
        raise ValueError(f"Y must hold M*N = {M * N} elements")
    if residual is not None:
        _need(residual, torch.float32, "residual")
        if residual.numel() != M * N:
            raise ValueError("residual must have M*N elements")
    _same_device(q.device, scale, X, Y, residual)
    ws = gemm_workspace(q.device, M, N, K)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().qz_gemm_w8_ws(q.data_ptr(), scale.data_ptr(), ng, X.data_ptr(),
                                             Y.data_ptr(), M, N, K, _ptr(residual),
                                             _ptr(ws), 0 if ws is None else ws.numel(),
                                             _stream_ptr(q.device)))
    return Y


def gemm_workspace(device, M: int, N: int, K: int):
    """Grow-only per-device workspace for the tensor-core GEMM (None when M < 2).

    The GEMM's activation split is stream-ordered on the current stream; two
    streams must not share this buffer concurrently.
    """
    import ctypes
    idx = ensure_device(device)
    need = ctypes.c_int64(0)
    _lib.check(_lib.load().qz_gemm_w8_workspace_bytes(M, N, K, ctypes.byref(need)))
    if need.value == 0:
        return None
    ws = _gemm_ws.get(idx)
    if ws is None or ws.numel() < need.value:
        ws = torch.empty(max(need.value, 1 << 20), dtype=torch.uint8,
                         device=torch.device("cuda", idx))
        _gemm_ws[idx] = ws
    return ws


def mlp_workspace(device) -> torch.Tensor:
    """Per-device grid-barrier words for the fused MLP (zeroed once)."""
    idx = ensure_device(device)
    ws = _mlp_ws.get(idx)
    if ws is None:
        nbytes = _lib.load().qz_mlp_workspace_bytes()
        ws = torch.zeros(nbytes // 4, dtype=torch.int32, device=torch.device("cuda", idx))
        _mlp_ws[idx] = ws
    return ws


def gemv_w4(q4, scale, x, y=None, residual=None):
    """int4 weights: y[n] = sum_g scale[n,g] sum_{j<G} x[gG+j] q[n,gG+j]
    (+ residual[n]), q4 uint8 [N, K/2] packed two weights per byte
    (quartz_b200.quantize.pack_int4)."""
    if not isinstance(q4, torch.Tensor) or q4.dtype != torch.uint8 or q4.dim() != 2:
        raise TypeError("q4 must be a 2-D uint8 CUDA tensor")
    if not q4.is_cuda or not q4.is_contiguous():
        raise ValueError("q4 must be a contiguous CUDA tensor")
    N, K = q4.shape[0], 2 * q4.shape[1]
    _need(scale, torch.float32, "scale", 2)
    if scale.shape[0] != N:
        raise ValueError("scale and q4 disagree on the number of rows")
    ng = scale.shape[1]
    ensure_device(q4.device)
    _need(x, torch.float32, "x")
    if x.numel() != K:
        raise ValueError(f"x has {x.numel()} elements, expected K={K}")
    if y is None:
        y = torch.empty(N, dtype=torch.float32, device=q4.device)
    _need(y, torch.float32, "y")
    if y.numel() != N:
        raise ValueError(f"y has {y.numel()} elements, expected N={N}")
    if residual is not None:
        _need(residual, torch.float32, "residual")
    _same_device(q4.device, scale, x, y, residual)
    with torch.cuda.device(q4.device):
        _lib.check(_lib.load().qz_gemv_w4(q4.data_ptr(), scale.data_ptr(), ng, x.data_ptr(),
                                          y.data_ptr(), N, K, _ptr(residual),
                                          _stream_ptr(q4.device)))
    return y


def fused_mlp(gu_q, gu_s, x, down_q, down_s, abuf=None, out=None, residual=None, norm_w=None,
              eps=1e-6):
    """out = down(silu(gate.x) * (up.x)) (+ residual) for one token (M = 1).
    With norm_w, of RMSNorm(x) * norm_w (normalised in the kernel)."""
    I2, H = gu_q.shape
    _, _, ng = _weights(gu_q, gu_s, "gu_q")
    Hd, I, ngd = _weights(down_q, down_s, "down_q")
    if I2 != 2 * I or Hd != H:
        raise ValueError(f"shape mismatch: gu_q {tuple(gu_q.shape)}, down_q {tuple(down_q.shape)}")
    dev = gu_q.device
    _need(x, torch.float32, "x")
    if x.numel() != H:
        raise ValueError(f"x has {x.numel()} elements, expected H={H}")
    if abuf is None:
        abuf = torch.empty(I, dtype=torch.float32, device=dev)
    if out is None:
        out = torch.empty(H, dtype=torch.float32, device=dev)
    _need(abuf, torch.float32, "abuf")
    _need(out, torch.float32, "out")
    if abuf.numel() != I or out.numel() != H:
        raise ValueError("abuf must have I elements and out H elements")
    if residual is not None:
        _need(residual, torch.float32, "residual")
        if residual.numel() != H:
            raise ValueError("residual must have H elements")
    _same_device(dev, gu_s, x, down_q, down_s, abuf, out, residual)
    ws = mlp_workspace(dev)
    if norm_w is not None:
        _need(norm_w, torch.float32, "norm_w", 1)
        if norm_w.numel() != H:
            raise ValueError("norm_w must have H elements")
        scratch = torch.empty(H, dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            _lib.check(_lib.load().qz_fused_mlp_decode_rmsnorm(
                gu_q.data_ptr(), gu_s.data_ptr(), ng, x.data_ptr(), norm_w.data_ptr(), float(eps),
                down_q.data_ptr(), down_s.data_ptr(), ngd, abuf.data_ptr(), out.data_ptr(),
                _ptr(residual), H, I, ws.data_ptr(), scratch.data_ptr(), _stream_ptr(dev)))
        return out
    with torch.cuda.device(dev):
        _lib.check(_lib.load().qz_fused_mlp_decode(
            gu_q.data_ptr(), gu_s.data_ptr(), ng, x.data_ptr(), down_q.data_ptr(),
            down_s.data_ptr(), ngd, abuf.data_ptr(), out.data_ptr(), _ptr(residual), H, I,
            ws.data_ptr(), _stream_ptr(dev)))
    return out


def silu_mul(gu, a=None):
    """a[m, i] = silu_clipped(gu[m, i]) * gu[m, I + i] for gu [M, 2I]."""
    _need(gu, torch.float32, "gu")
    ensure_device(gu.device)
    M = gu.numel() // gu.shape[-1]
    I2 = gu.shape[-1]
    if I2 % 2:
        raise ValueError("gu's last dimension must be even")
    I = I2 // 2
    if a is None:
        a = torch.empty((*gu.shape[:-1], I), dtype=torch.float32, device=gu.device)
    _need(a, torch.float32, "a")
    if a.numel() != M * I:
        raise ValueError(f"a must hold M*I = {M * I} elements")
    _same_device(gu.device, a)
    with torch.cuda.device(gu.device):
        _lib.check(_lib.load().qz_silu_mul(gu.data_ptr(), a.data_ptr(), M, I,
                                           _stream_ptr(gu.device)))
    return a


def status(clear: bool = False, device=None):
    """Device status word {error bits, first site, its block, count} (synchronises)."""
    idx = ensure_device(device)
    with torch.cuda.device(idx):
        return _lib.device_status(clear)


def check_status(device=None) -> None:
    """Raise if any kernel on the device reported a failed wait; clears the word."""
    bits, site, block, count = status(clear=True, device=device)
    if bits:
        raise _lib.QuartzError(
            f"device kernels reported {count} failed wait(s): bits=0x{bits:x} "
            f"first site=0x{site:x} block={block}")


# ---------------------------------------------------------------------------
# decode-step glue
# ---------------------------------------------------------------------------

_attn_ws: dict[int, torch.Tensor] = {}
_argmax_keys: dict[int, torch.Tensor] = {}


def embed_gather(q, scale, ids, out=None):
    """out[m, :] = q[ids[m], :] * scale[ids[m], group] (int64 ids on the device)."""
    V, H, ng = _weights(q, scale)
    ensure_device(q.device)
    _need(ids, torch.int64, "ids")
    M = ids.numel()
    if out is None:
        out = torch.empty((M, H), dtype=torch.float32, device=q.device)
    _need(out, torch.float32, "out")
    if out.numel() != M * H:
        raise ValueError(f"out must hold M*H = {M * H} elements")
    _same_device(q.device, scale, ids, out)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().qz_embed_gather(q.data_ptr(), scale.data_ptr(), ng, ids.data_ptr(),
                                               M, V, H, out.data_ptr(), _stream_ptr(q.device)))
    return out


def rmsnorm(x, w, eps=1e-6, out=None):
    """Row-wise x / sqrt(mean(x^2) + eps) * w over the last dimension."""
    _need(x, torch.float32, "x")
    _need(w, torch.float32, "w", 1)
    ensure_device(x.device)
    n = x.shape[-1]
    if w.numel() != n:
        raise ValueError(f"w has {w.numel()} elements, rows have {n}")
    rows = x.numel() // n if n else 0
    if out is None:
        out = torch.empty_like(x)
    _need(out, torch.float32, "out")
    if out.numel() != x.numel():
        raise ValueError("out must match x")
    _same_device(x.device, w, out)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().qz_rmsnorm(x.data_ptr(), w.data_ptr(), out.data_ptr(), rows, n,
                                          float(eps), _stream_ptr(x.device)))
    return out


def _cache_dims(kc, vc):
    _need(kc, torch.float32, "k_cache", 3)
    _need(vc, torch.float32, "v_cache", 3)
    if kc.shape != vc.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    return kc.shape   # (n_kv, max_ctx, head_dim)


def qk_rope(qkv, inv_freq, k_cache, v_cache, n_heads, pos0=0, pos_dev=None, q_norm=None,
            k_norm=None, eps=1e-6, q_out=None):
    """Split qkv [M, (nq + 2 nkv) hd] into q (normed, rotated; returned as [M, nq hd]) and the
    cache rows at positions pos0 + m (or *pos_dev + m)."""
    nkv, max_ctx, hd = _cache_dims(k_cache, v_cache)
    _need(qkv, torch.float32, "qkv")
    _need(inv_freq, torch.float32, "inv_freq", 1)
    ensure_device(qkv.device)
    width = (n_heads + 2 * nkv) * hd
    if qkv.shape[-1] != width:
        raise ValueError(f"qkv rows must have {width} elements")
    if inv_freq.numel() != hd // 2:
        raise ValueError("inv_freq must have head_dim / 2 elements")
    M = qkv.numel() // width
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _need(t, torch.float32, name, 1)
            if t.numel() != hd:
                raise ValueError(f"{name} must have head_dim elements")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("pass both q_norm and k_norm or neither")
    if pos_dev is not None:
        _need(pos_dev, torch.int64, "pos_dev")
    if q_out is None:
        q_out = torch.empty((M, n_heads * hd), dtype=torch.float32, device=qkv.device)
    _need(q_out, torch.float32, "q_out")
    if q_out.numel() != M * n_heads * hd:
        raise ValueError("q_out must hold M * n_heads * head_dim elements")
    _same_device(qkv.device, inv_freq, k_cache, v_cache, q_norm, k_norm, pos_dev, q_out)
    with torch.cuda.device(qkv.device):
        _lib.check(_lib.load().qz_qk_rope(
            qkv.data_ptr(), _ptr(q_norm), _ptr(k_norm), inv_freq.data_ptr(), q_out.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), M, n_heads, nkv, hd, max_ctx, int(pos0),
            _ptr(pos_dev), float(eps), _stream_ptr(qkv.device)))
    return q_out


def attention_workspace(device, n_heads: int, n_kv: int, head_dim: int, max_ctx: int
                        ) -> torch.Tensor:
    """Grow-only per-device workspace of the decode attention (zeroed when made;
    the kernels leave it zeroed where it must be)."""
    import ctypes
    idx = ensure_device(device)
    need = ctypes.c_int64(0)
    with torch.cuda.device(idx):
        _lib.check(_lib.load().qz_attention_decode_workspace_bytes(n_heads, n_kv, head_dim,
                                                                   max_ctx, ctypes.byref(need)))
    ws = _attn_ws.get(idx)
    if ws is None or ws.numel() < need.value:
        ws = torch.zeros(need.value, dtype=torch.uint8, device=torch.device("cuda", idx))
        _attn_ws[idx] = ws
    return ws


def attention_decode(q, k_cache, v_cache, T=None, T_dev=None, t_offset=0, scale=None, out=None,
                     workspace=None):
    """softmax(q K^T * scale) V for one query row per head over cache positions [0, T)
    (T = *T_dev + t_offset when T_dev is given). q: [n_heads * head_dim]."""
    nkv, max_ctx, hd = _cache_dims(k_cache, v_cache)
    _need(q, torch.float32, "q")
    ensure_device(q.device)
    if q.numel() % hd:
        raise ValueError("q must hold n_heads * head_dim elements")
    nq = q.numel() // hd
    if (T is None) == (T_dev is None):
        raise ValueError("pass exactly one of T and T_dev")
    if T_dev is not None:
        _need(T_dev, torch.int64, "T_dev")
    scale = hd ** -0.5 if scale is None else scale
    if out is None:
        out = torch.empty(nq * hd, dtype=torch.float32, device=q.device)
    _need(out, torch.float32, "out")
    if out.numel() != nq * hd:
        raise ValueError("out must hold n_heads * head_dim elements")
    ws = workspace if workspace is not None else attention_workspace(q.device, nq, nkv, hd,
                                                                      max_ctx)
    _same_device(q.device, k_cache, v_cache, T_dev, out, ws)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().qz_attention_decode(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), nq, nkv, hd,
            max_ctx, 0 if T is None else int(T), _ptr(T_dev), int(t_offset), float(scale),
            ws.data_ptr(), ws.numel(), _stream_ptr(q.device)))
    return out


def attention_decode_qkv(qkv, inv_freq, k_cache, v_cache, n_heads, pos0=0, pos_dev=None,
                         q_norm=None, k_norm=None, eps=1e-6, scale=None, out=None,
                         workspace=None):
    """The attention block of one decode token from its projection row qkv
    [(nq + 2 nkv) hd]: q/k norm (Qwen3), RoPE, k/v append at position pos0
    (or *pos_dev), attention over positions [0, pos]. Returns [nq * hd]."""
    nkv, max_ctx, hd = _cache_dims(k_cache, v_cache)
    _need(qkv, torch.float32, "qkv")
    _need(inv_freq, torch.float32, "inv_freq", 1)
    ensure_device(qkv.device)
    if qkv.numel() != (n_heads + 2 * nkv) * hd:
        raise ValueError(f"qkv must hold (n_heads + 2 n_kv) * head_dim elements")
    if inv_freq.numel() != hd // 2:
        raise ValueError("inv_freq must have head_dim / 2 elements")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("pass both q_norm and k_norm or neither")
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _need(t, torch.float32, name, 1)
            if t.numel() != hd:
                raise ValueError(f"{name} must have head_dim elements")
    if pos_dev is not None:
        _need(pos_dev, torch.int64, "pos_dev")
    scale = hd ** -0.5 if scale is None else scale
    if out is None:
        out = torch.empty(n_heads * hd, dtype=torch.float32, device=qkv.device)
    _need(out, torch.float32, "out")
    if out.numel() != n_heads * hd:
        raise ValueError("out must hold n_heads * head_dim elements")
    ws = workspace if workspace is not None else attention_workspace(qkv.device, n_heads, nkv, hd,
                                                                      max_ctx)
    _same_device(qkv.device, inv_freq, k_cache, v_cache, q_norm, k_norm, pos_dev, out, ws)
    with torch.cuda.device(qkv.device):
        _lib.check(_lib.load().qz_attention_decode_qkv(
            qkv.data_ptr(), _ptr(q_norm), _ptr(k_norm), inv_freq.data_ptr(), k_cache.data_ptr(),
            v_cache.data_ptr(), out.data_ptr(), n_heads, nkv, hd, max_ctx, int(pos0),
            _ptr(pos_dev), float(eps), float(scale), ws.data_ptr(), ws.numel(),
            _stream_ptr(qkv.device)))
    return out


def attention_prefill(q, k_cache, v_cache, pos0, scale=None, out=None):
    """Causal attention of query rows q [M, n_heads * head_dim] at positions pos0 + m."""
    nkv, max_ctx, hd = _cache_dims(k_cache, v_cache)
    _need(q, torch.float32, "q", 2)
    ensure_device(q.device)
    M, width = q.shape
    if width % hd:
        raise ValueError("q rows must hold n_heads * head_dim elements")
    nq = width // hd
    scale = hd ** -0.5 if scale is None else scale
    if out is None:
        out = torch.empty_like(q)
    _need(out, torch.float32, "out")
    if out.numel() != q.numel():
        raise ValueError("out must match q")
    _same_device(q.device, k_cache, v_cache, out)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().qz_attention_prefill(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), M, nq, nkv, hd,
            max_ctx, int(pos0), float(scale), _stream_ptr(q.device)))
    return out


def argmax_keys(device, M: int) -> torch.Tensor:
    """Per-device zeroed uint64 scratch for argmax (kept zero between calls)."""
    idx = ensure_device(device)
    keys = _argmax_keys.get(idx)
    if keys is None or keys.numel() < M:
        keys = torch.zeros(max(M, 64), dtype=torch.int64, device=torch.device("cuda", idx))
        _argmax_keys[idx] = keys
    return keys


def argmax(logits, tokens=None, pos_dev=None, pos_step=0, keys=None):
    """Greedy token per row of logits [M, V] (first index of the maximum)."""
    _need(logits, torch.float32, "logits")
    ensure_device(logits.device)
    V = logits.shape[-1]
    M = logits.numel() // V
    if tokens is None:
        tokens = torch.empty(M, dtype=torch.int64, device=logits.device)
    _need(tokens, torch.int64, "tokens")
    if tokens.numel() != M:
        raise ValueError("tokens must have one element per row")
    if pos_dev is not None:
        _need(pos_dev, torch.int64, "pos_dev")
    keys = keys if keys is not None else argmax_keys(logits.device, M)
    _same_device(logits.device, tokens, pos_dev, keys)
    with torch.cuda.device(logits.device):
        _lib.check(_lib.load().qz_argmax(logits.data_ptr(), M, V, keys.data_ptr(),
                                         tokens.data_ptr(), _ptr(pos_dev), int(pos_step),
                                         _stream_ptr(logits.device)))
    return tokens


# ---------------------------------------------------------------------------
# paged 4-bit KV cache
# ---------------------------------------------------------------------------

KV4_PAGE_SIZES = (16, 32, 64, 128, 256)
KV4_HEAD_DIMS = (64, 128)
_KV4_DTYPES = {torch.float32: _lib.QZ_F32, torch.bfloat16: _lib.QZ_BF16,
               torch.float16: _lib.QZ_F16}
_kv4_ws: dict[tuple[int, int], torch.Tensor] = {}
_kv4_ws_need: dict[tuple, int] = {}


class KV4Plan(NamedTuple):
    """What kv4_plan returns: int64 tensors. Rows of request b are
    cu_rows[b] .. cu_rows[b + 1] - 1; lens and used are the successors of the
    arguments; slots and positions are per row (-1: no place in the cache, and
    rows behind the last request's)."""
    cu_rows: torch.Tensor
    lens: torch.Tensor
    used: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor


class _on:
    """Makes a device current for a library call (nothing to do in the usual case
    that it is)."""
    __slots__ = ("idx", "prev")

    def __init__(self, idx: int):
        self.idx = idx

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.prev != self.idx:
            torch.cuda.set_device(self.idx)

    def __exit__(self, *exc):
        if self.prev != self.idx:
            torch.cuda.set_device(self.prev)


def _arg(t, dtype, name: str, ndim: int, idx: int) -> None:
    """A contiguous tensor of dtype and ndim on GPU idx: one condition in the usual
    case, _need and _same_device to say what is wrong. (These calls take a few
    microseconds of GPU time at decode sizes, about what their checks do.)"""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.dim() == ndim
            and t.get_device() == idx and t.is_contiguous()):
        _need(t, dtype, name, ndim)
        _same_device(torch.device("cuda", idx), t)


def _home(t, name: str) -> int:
    """The index of the GPU a tensor is on, which the call then runs on."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    idx = t.get_device()
    if idx not in _ready_devices:
        ensure_device(idx)
    return idx


def kv4_block_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one page of one kv head: K and V codes and their (s, z) pairs."""
    if page_size not in KV4_PAGE_SIZES:
        raise ValueError(f"page_size must be one of {KV4_PAGE_SIZES}, got {page_size}")
    if head_dim not in KV4_HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {KV4_HEAD_DIMS}, got {head_dim}")
    return page_size * (head_dim + 8)


def kv4_pool(pages: int, n_kv: int, head_dim: int, page_size: int, device=None) -> torch.Tensor:
    """The zeroed pool of one layer, uint8 [pages, n_kv, page_size * (head_dim + 8)]."""
    nbytes = kv4_block_bytes(page_size, head_dim)
    return torch.zeros((pages, n_kv, nbytes), dtype=torch.uint8,
                       device=torch.device("cuda", ensure_device(device)))


_kv4_ps: dict[tuple[int, int], int] = {
    (qz_ps * (qz_hd + 8), qz_hd): qz_ps for qz_ps in KV4_PAGE_SIZES for qz_hd in KV4_HEAD_DIMS}


def _kv4_page_size(pool: torch.Tensor, head_dim: int, idx: int) -> int:
    """The page size of a pool (checked against head_dim)."""
    _arg(pool, torch.uint8, "pool", 3, idx)
    ps = _kv4_ps.get((pool.shape[2], head_dim))
    if ps is None:
        if head_dim not in KV4_HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {KV4_HEAD_DIMS}, got {head_dim}")
        raise ValueError(f"pool blocks of {pool.shape[2]} bytes are no pages of head_dim {head_dim}")
    return ps


def _kv4_rows(t: torch.Tensor, name: str, idx: int) -> tuple[int, int, int]:
    """Shape of rows [n, heads, head_dim] on GPU idx, any strides with contiguous
    head_dim."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in _KV4_DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != 3:
        raise ValueError(f"{name} must be [rows, heads, head_dim], got shape {tuple(t.shape)}")
    if t.get_device() != idx:
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        _same_device(torch.device("cuda", idx), t)
    if t.stride(2) != 1:
        raise ValueError(f"{name} must be contiguous along head_dim")
    return t.shape


def kv4_plan(lens, new_rows, block_table, free_pages, used, page_size, rows, lens_out=None,
             used_out=None) -> KV4Plan:
    """Block tables and slot maps of one step, built on the GPU from request lengths.

    lens, new_rows: int64 [B], the positions each request holds and the rows
    that join it now (B <= 4096). block_table: int32 [B, W], written in place
    (new entries only). free_pages: int32 [F] in the order they are handed out,
    used: int64 [1], how many of them are taken. rows: the row capacity of this
    step (padding included). A request whose rows do not fit `rows`, whose pages
    do not fit W, or for which the free pages do not last (counted in order)
    keeps its length and gets slots -1. lens_out / used_out may be lens / used
    themselves (a step captured in a CUDA graph then advances them)."""
    if _fast is not None:
        r = _fast.plan(lens, new_rows, block_table, free_pages, used, page_size, rows, lens_out,
                       used_out)
        if r is not None:
            return KV4Plan._make(r)
    idx = _home(lens, "lens")
    _arg(lens, torch.int64, "lens", 1, idx)
    _arg(new_rows, torch.int64, "new_rows", 1, idx)
    _arg(block_table, torch.int32, "block_table", 2, idx)
    _arg(free_pages, torch.int32, "free_pages", 1, idx)
    _arg(used, torch.int64, "used", 1, idx)
    B, W = block_table.shape
    rows = int(rows)
    if lens.numel() != B or new_rows.numel() != B:
        raise ValueError(f"lens and new_rows must have one element per table row ({B})")
    if used.numel() != 1:
        raise ValueError("used must have one element")
    if rows < 0:
        raise ValueError("rows must not be negative")
    buf = torch.empty(2 * B + 2 + 2 * rows, dtype=torch.int64, device=lens.device)
    cu, lo, uo, slots, positions = torch.unsafe_split_with_sizes(buf, (B + 1, B, 1, rows, rows))
    if lens_out is not None:
        _arg(lens_out, torch.int64, "lens_out", 1, idx)
        if lens_out.numel() != B:
            raise ValueError(f"lens_out must have {B} elements")
        lo = lens_out
    if used_out is not None:
        _arg(used_out, torch.int64, "used_out", 1, idx)
        if used_out.numel() != 1:
            raise ValueError("used_out must have one element")
        uo = used_out
    at = buf.data_ptr()                    # the parts lie one behind the other
    with _on(idx):
        _lib.check(_lib.load().qz_kv4_plan(
            lens.data_ptr(), new_rows.data_ptr(), B, block_table.data_ptr(), W,
            free_pages.data_ptr(), free_pages.numel(), used.data_ptr(), int(page_size), rows, at,
            lo.data_ptr(), uo.data_ptr(), at + 8 * (2 * B + 2), at + 8 * (2 * B + 2 + rows),
            _stream_ptr(lens.device)))
    return KV4Plan(cu, lo, uo, slots, positions)


def kv4_append(k, v, pool, slots) -> None:
    """Quantise rows k, v [n, n_kv, hd] (float32, bfloat16 or float16; hd
    contiguous, other strides free) to 4 bits and store row r at slots[r]
    (int64 [n]; a slot outside the pool stores nothing). Each row of a kv head
    keeps its own bf16 step and zero; a row with a non-finite value reads back
    as NaN. A slot must not appear twice in one call."""
    if _fast is not None and _fast.append(k, v, pool, slots):
        return
    if not (isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise TypeError("k and v must be torch.Tensors")
    idx = _home(pool, "pool")
    n, nkv, hd = _kv4_rows(k, "k", idx)
    _kv4_rows(v, "v", idx)
    if k.shape != v.shape or k.dtype is not v.dtype:
        raise ValueError("k and v must have the same shape and dtype")
    ps = _kv4_page_size(pool, hd, idx)
    if pool.shape[1] != nkv:
        raise ValueError(f"pool has {pool.shape[1]} kv heads, k has {nkv}")
    _arg(slots, torch.int64, "slots", 1, idx)
    if slots.numel() != n:
        raise ValueError(f"slots must have one element per row ({n})")
    ks, vs = k.stride(), v.stride()
    with _on(idx):
        _lib.check(_lib.load().qz_kv4_append(
            k.data_ptr(), v.data_ptr(), _KV4_DTYPES[k.dtype], ks[0], ks[1], vs[0], vs[1], n, nkv,
            hd, pool.data_ptr(), pool.shape[0], ps, slots.data_ptr(), _stream_ptr(pool.device)))


def kv4_gather(pool, slots, head_dim, out=None):
    """(k, v) fp32 [n, n_kv, head_dim]: the values at slots (int64 [n]); zeros
    for a slot outside the pool. out: a pair of contiguous tensors to write."""
    if _fast is not None and out is None:
        r = _fast.gather(pool, slots, head_dim)
        if r is not None:
            return r
    idx = _home(pool, "pool")
    hd = int(head_dim)
    ps = _kv4_page_size(pool, hd, idx)
    _arg(slots, torch.int64, "slots", 1, idx)
    n, nkv = slots.numel(), pool.shape[1]
    if out is None:
        k = torch.empty((n, nkv, hd), dtype=torch.float32, device=pool.device)
        v = torch.empty_like(k)
    else:
        k, v = out
        for t, name in ((k, "out[0]"), (v, "out[1]")):
            _arg(t, torch.float32, name, 3, idx)
            if tuple(t.shape) != (n, nkv, hd):
                raise ValueError(f"{name} must be [{n}, {nkv}, {hd}], got {tuple(t.shape)}")
    with _on(idx):
        _lib.check(_lib.load().qz_kv4_gather(
            pool.data_ptr(), pool.shape[0], ps, nkv, hd, slots.data_ptr(), n, k.data_ptr(),
            v.data_ptr(), _stream_ptr(pool.device)))
    return k, v


def qk_rope_kv4(qkv, inv_freq, positions, pool, slots, n_heads, q_norm=None, k_norm=None,
                eps=1e-6, q_out=None):
    """Split projection rows qkv [M, (nq + 2 nkv) hd] (fp32) into q, normed and rotated at
    positions [M] (returned as [M, nq, hd]), and the k and v rows, which are stored
    in the paged cache at slots [M] as kv4_append would."""
    idx = _home(pool, "pool")
    _arg(inv_freq, torch.float32, "inv_freq", 1, idx)
    hd = 2 * inv_freq.numel()
    ps = _kv4_page_size(pool, hd, idx)
    nkv = pool.shape[1]
    _arg(qkv, torch.float32, "qkv", 2, idx)
    _arg(positions, torch.int64, "positions", 1, idx)
    _arg(slots, torch.int64, "slots", 1, idx)
    M = qkv.shape[0]
    if qkv.shape[1] != (n_heads + 2 * nkv) * hd:
        raise ValueError(f"qkv rows must have {(n_heads + 2 * nkv) * hd} elements")
    if positions.numel() != M or slots.numel() != M:
        raise ValueError(f"positions and slots must have one element per row ({M})")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("pass both q_norm and k_norm or neither")
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _arg(t, torch.float32, name, 1, idx)
            if t.numel() != hd:
                raise ValueError(f"{name} must have head_dim elements")
    if q_out is None:
        q_out = torch.empty((M, n_heads, hd), dtype=torch.float32, device=pool.device)
    elif not (isinstance(q_out, torch.Tensor) and q_out.dtype is torch.float32
              and q_out.get_device() == idx and q_out.is_contiguous()):
        _need(q_out, torch.float32, "q_out")
        _same_device(pool.device, q_out)
    if q_out.numel() != M * n_heads * hd:
        raise ValueError("q_out must hold M * n_heads * head_dim elements")
    with _on(idx):
        _lib.check(_lib.load().qz_qk_rope_kv4(
            qkv.data_ptr(), _ptr(q_norm), _ptr(k_norm), inv_freq.data_ptr(), q_out.data_ptr(), M,
            n_heads, nkv, hd, positions.data_ptr(), pool.data_ptr(), pool.shape[0], ps,
            slots.data_ptr(), float(eps), _stream_ptr(pool.device)))
    return q_out


def kv4_attention_workspace(device, n_heads: int, n_kv: int, head_dim: int, max_rows: int = 1
                            ) -> torch.Tensor:
    """A new zeroed workspace of kv4_attention for calls with up to max_rows rows
    per request. The calls leave it ready for the next one; calls that may
    overlap on the GPU (other streams, graphs replayed side by side) must not
    share one."""
    idx = ensure_device(device)
    return torch.zeros(_kv4_ws_bytes(idx, n_heads, n_kv, head_dim, max_rows), dtype=torch.uint8,
                       device=torch.device("cuda", idx))


def _kv4_ws_bytes(idx: int, nq: int, nkv: int, hd: int, max_rows: int) -> int:
    key = (idx, nq, nkv, hd, max_rows)
    need = _kv4_ws_need.get(key)
    if need is None:
        b = ctypes.c_int64(0)
        with _on(idx):
            _lib.check(_lib.load().qz_kv4_attention_workspace_bytes(nq, nkv, hd, max_rows,
                                                                    ctypes.byref(b)))
        if len(_kv4_ws_need) > 4096:
            _kv4_ws_need.clear()
        need = _kv4_ws_need[key] = b.value
    return need


def _kv4_default_ws(idx: int, stream: int, need: int) -> torch.Tensor:
    """The workspace of a call that brings none: one per device and stream. A call
    under stream capture gets its own, so that two graphs (or a graph and eager
    calls) never share one."""
    def made():
        ws = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", idx))
        ws[:_lib.QZ_KV4_WORKSPACE_HEAD].zero_()
        return ws

    if torch._C._cuda_isCurrentStreamCapturing():
        return made()
    ws = _kv4_ws.get((idx, stream))
    if ws is None or ws.numel() < need:
        ws = made()
        _kv4_ws[idx, stream] = ws
        if _fast is not None:
            _fast.workspace(idx, stream, ws.data_ptr(), ws.numel())
    return ws


def kv4_attention(q, pool, block_table, lens, cu_rows=None, max_rows=None, scale=None, out=None,
                  workspace=None):
    """softmax(scale * q K^T) V of query rows over the paged 4-bit cache.

    q: [n, n_heads, hd] (float32, bfloat16 or float16; hd contiguous). Rows
    cu_rows[b] .. cu_rows[b + 1] - 1 are the last rows of request b, whose
    lens[b] positions (int64 [B], this step's included) lie in the pages
    block_table[b] (int32 [B, W]); each sees the positions up to its own, and
    one that sees none gives zeros. cu_rows (int64 [B + 1]) None: row b is
    request b's (lens beyond the n rows are not used). max_rows: the most rows a
    request has (a host number; rows of a request with more are not computed);
    n unless given, 1 without cu_rows. scale: hd ** -0.5 unless given. Returns
    out (q's dtype); rows that are not computed are left as they were, and are
    zeros in an output that the call makes. out may be q itself, but must not
    overlap it otherwise. n, B and max_rows choose between two kernels, whose
    results differ by rounding."""
    if _fast is not None:
        r = _fast.attention(q, pool, block_table, lens, cu_rows, max_rows, scale, out, workspace)
        if r is not None:
            return r
    idx = _home(pool, "pool")
    n, nq, hd = _kv4_rows(q, "q", idx)
    ps = _kv4_page_size(pool, hd, idx)
    pages, nkv = pool.shape[0], pool.shape[1]
    _arg(block_table, torch.int32, "block_table", 2, idx)
    _arg(lens, torch.int64, "lens", 1, idx)
    B, W = block_table.shape
    if lens.numel() != B:
        raise ValueError(f"lens must have one element per table row ({B})")
    max_rows = (1 if cu_rows is None else max(1, n)) if max_rows is None else int(max_rows)
    if cu_rows is not None:
        _arg(cu_rows, torch.int64, "cu_rows", 1, idx)
        if cu_rows.numel() != B + 1:
            raise ValueError(f"cu_rows must have {B + 1} elements")
    if nq % nkv:
        raise ValueError(f"{nq} query heads are no multiple of {nkv} kv heads")
    scale = hd ** -0.5 if scale is None else float(scale)
    qs = q.stride()
    if out is None:
        # which rows are computed is in cu_rows, on the GPU
        make = torch.empty if cu_rows is None and n <= B else torch.zeros
        out = make((n, nq, hd), dtype=q.dtype, device=pool.device)
    else:
        _kv4_rows(out, "out", idx)
        if out.shape != q.shape or out.dtype is not q.dtype:
            raise ValueError("out must have q's shape and dtype")
    os = out.stride()
    if not ((nq == 1 or os[1] >= hd) and (n == 1 or os[0] >= (nq - 1) * os[1] + hd)
            or (n == 1 or os[0] >= hd) and (nq == 1 or os[1] >= (n - 1) * os[0] + hd)):
        raise ValueError("out's rows and heads must not overlap")
    with _on(idx):
        st = _stream_ptr(pool.device)
        if workspace is None:
            workspace = _kv4_default_ws(idx, st, _kv4_ws_bytes(idx, nq, nkv, hd, max_rows))
        else:
            _arg(workspace, torch.uint8, "workspace", 1, idx)
        _lib.check(_lib.load().qz_kv4_attention(
            q.data_ptr(), _KV4_DTYPES[q.dtype], qs[0], qs[1], out.data_ptr(), os[0], os[1],
            pool.data_ptr(), pages, ps, block_table.data_ptr(), W, lens.data_ptr(), _ptr(cu_rows),
            B, n, max_rows, nq, nkv, hd, scale, workspace.data_ptr(), workspace.numel(), st))
    return out
