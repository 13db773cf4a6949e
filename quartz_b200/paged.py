"""All-int8 greedy decoding of requests of uneven length over a paged 4-bit KV cache.

quartz decodes a batch in lockstep over one growing cache (quartz/models/
common.py:79-88, quartz/cache.py:26-46). ``PagedEngine`` keeps requests that
start, grow and end independently: their K and V rows live in pages of a shared
pool, quantised to 4 bits with a step and a zero per row, and every step's block
tables, slots and positions are built on the GPU (``device.kv4_plan``). A layer
of a step of N rows is

    RMSNorm + q/k/v GEMM -> qk_rope_kv4 (q/k norm, RoPE, 4-bit append)
    -> kv4_attention -> o GEMM + residual -> RMSNorm + gate/up GEMM
    -> silu-mul + down GEMM + residual

with the kernels of ``DecodeEngine`` around the paged ones. A decode step (one
row per request) is captured in a CUDA graph for each number of running
requests; the plan advances lengths and the page cursor in place, so a replay
needs nothing from the host. The host only keeps lengths (which it can count)
and compacts the batch when a request ends.

Differences of result from ``DecodeEngine``: K and V are 4-bit (13 to 14 % of
the fp32 cache's bytes), so logits differ by the quantisation.
"""

from __future__ import annotations

import ctypes
from typing import Iterable, Mapping, Sequence

import torch

from . import _lib, device as qd
from .decode import _Int8Weights, quartz_checkpoint
from .model import ModelSpec


class PagedEngine(_Int8Weights):
    """Greedy decoder of up to max_batch requests over `pages` pages of 4-bit K/V.

    weights and norms as DecodeEngine's. max_ctx: the longest a request may get
    (prompt and generated tokens); max_rows: prompt rows processed in one step;
    page_size: positions per page (16 .. 256, a power of two)."""

    def __init__(self, spec: ModelSpec, int8_weights: Mapping | Iterable, norms: Mapping, *,
                 pages: int, max_ctx: int, max_batch: int = 16, page_size: int = 32,
                 max_rows: int = 512, device=None, fold_norms: bool = True):
        qd.kv4_block_bytes(page_size, spec.head_dim)      # refuses what the kernels do not take
        if pages < 1 or max_batch < 1 or max_rows < 1 or max_ctx < 1:
            raise ValueError("pages, max_ctx, max_batch and max_rows must be >= 1")
        if max_batch > 4096:
            raise ValueError("at most 4096 requests run at once")
        self.spec = spec
        self.dev = torch.device("cuda", qd.ensure_device(device))
        self.lib = _lib.load()
        self.page_size, self.pages = int(page_size), int(pages)
        self.max_ctx, self.max_batch = int(max_ctx), int(max_batch)
        self.max_rows = max(int(max_rows), self.max_batch, 2)
        self.fold_norms = bool(fold_norms)
        self._load_weights(int8_weights, norms)
        S, dev = spec, self.dev
        H, hd, Mx = S.hidden, S.head_dim, self.max_rows
        width = -(-self.max_ctx // self.page_size)
        self.pool = torch.zeros((S.layers, self.pages, S.n_kv,
                                 qd.kv4_block_bytes(self.page_size, hd)), dtype=torch.uint8,
                                device=dev)
        i64 = dict(dtype=torch.int64, device=dev)
        self.table = torch.full((self.max_batch, width), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(self.max_batch, **i64)
        self.free_pages = torch.arange(self.pages, dtype=torch.int32, device=dev)
        self.used = torch.zeros(1, **i64)
        self.one = torch.ones(self.max_batch, **i64)
        f32 = dict(dtype=torch.float32, device=dev)
        self.h_a, self.h_b, self.xn = (torch.zeros((Mx, H), **f32) for _ in range(3))
        self.qkv = torch.zeros((Mx, S.qkv_rows), **f32)
        self.qo, self.ao = (torch.zeros((Mx, S.n_heads, hd), **f32) for _ in range(2))
        self.gu = torch.zeros((Mx, 2 * S.inter), **f32)
        self.act = torch.zeros((Mx, S.inter), **f32)
        rows = max(2, self.max_batch)
        self.h_last = torch.zeros((rows, H), **f32)
        self.logits = torch.zeros((rows, S.vocab), **f32)
        self.keys = torch.zeros(rows, **i64)
        self.tok = torch.zeros(rows, **i64)
        self.ids = torch.zeros(Mx, **i64)
        need = 0
        for M in (Mx, rows):
            for N, K in ((S.qkv_rows, H), (H, S.n_heads * hd), (2 * S.inter, H), (H, S.inter),
                         (S.vocab, H)):
                b = ctypes.c_int64(0)
                _lib.check(self.lib.qz_gemm_w8_workspace_bytes(M, N, K, ctypes.byref(b)))
                need = max(need, b.value)
        self.gemm_ws = torch.empty(need, dtype=torch.uint8, device=dev)
        sizes = [qd.kv4_attention_workspace(dev, S.n_heads, S.n_kv, hd, m).numel() for m in (1, Mx)]
        self.attn_ws = torch.zeros(max(sizes), dtype=torch.uint8, device=dev)
        # host mirror of the running requests, in the order of the table's rows
        self._ids: list[int] = []        # request id
        self._len: list[int] = []        # positions held
        self._next: list[int] = []       # the token that its next step takes
        self._held: list[list[int]] = []  # tokens emitted during other requests' generate
        self._used = 0                   # pages handed out
        self._serial = 0
        self._graphs: dict[int, torch.cuda.CUDAGraph] = {}

    @classmethod
    def from_quartz(cls, net, **kw) -> "PagedEngine":
        """An engine on the int8 weights of a quantised quartz model (see
        decode.quartz_checkpoint); keyword arguments as the constructor's."""
        spec, int8, norms = quartz_checkpoint(net)
        return cls(spec, int8, norms, **kw)

    # ---------------------------------------------------------------- queries
    @property
    def running(self) -> list[int]:
        """Ids of the running requests."""
        return list(self._ids)

    @property
    def free(self) -> int:
        """Pages that no request holds."""
        return self.pages - self._used

    def length(self, request: int) -> int:
        """Positions a request holds in the cache."""
        return self._len[self._row(request)]

    def _row(self, request: int) -> int:
        try:
            return self._ids.index(request)
        except ValueError:
            raise KeyError(f"no running request {request}") from None

    def _pages_of(self, positions: int) -> int:
        return -(-positions // self.page_size)

    def kv(self, request: int, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(k, v) fp32 [positions, n_kv, head_dim] that a request's cache stands for."""
        row = self._row(request)
        if not 0 <= layer < self.spec.layers:
            raise IndexError("no such layer")
        p = torch.arange(self._len[row], device=self.dev)
        slots = self.table[row].long()[p // self.page_size] * self.page_size + p % self.page_size
        return qd.kv4_gather(self.pool[layer], slots, self.spec.head_dim)

    # ------------------------------------------------------------ the layers
    def _forward(self, plan: qd.KV4Plan, B: int, M: int, max_rows: int, st: int) -> None:
        """ids [M] -> h_a [M, H] after all layers; appends to the cache of the
        first B requests."""
        S, lib, chk = self.spec, self.lib, _lib.check
        H, hd, nq, I = S.hidden, S.head_dim, S.n_heads, S.inter
        p = lambda t: t.data_ptr()  # noqa: E731
        h_a, h_b = p(self.h_a), p(self.h_b)
        ws, wsb = p(self.gemm_ws), self.gemm_ws.numel()
        chk(lib.qz_embed_gather(p(self.embed_q), p(self.embed_s), self.embed_s.shape[1],
                                p(self.ids), M, S.vocab, H, h_a, st))
        q, ao = self.qo[:M], self.ao[:M]
        table, lens = self.table[:B], self.lens[:B]
        for li, L in enumerate(self.layers):
            self._gemm_act(L.qkv_q, L.qkv_s, h_a, _lib.QZ_ACT_RMSNORM, p(L.in_w), p(self.qkv), M,
                           S.qkv_rows, H, None, st)
            qd.qk_rope_kv4(self.qkv[:M], self.inv_freq, plan.positions, self.pool[li], plan.slots,
                           nq, L.qn_w, L.kn_w, S.eps, q_out=q)
            qd.kv4_attention(q, self.pool[li], table, lens, cu_rows=plan.cu_rows,
                             max_rows=max_rows, scale=self.attn_scale, out=ao,
                             workspace=self.attn_ws)
            chk(lib.qz_gemm_w8_ws(p(L.o_q), p(L.o_s), L.o_s.shape[1], p(ao), h_b, M, H, nq * hd,
                                  h_a, ws, wsb, st))
            self._gemm_act(L.gu_q, L.gu_s, h_b, _lib.QZ_ACT_RMSNORM, p(L.post_w), p(self.gu), M,
                           2 * I, H, None, st)
            self._gemm_act(L.down_q, L.down_s, p(self.gu), _lib.QZ_ACT_SILU_MUL, None, h_a, M, H,
                           I, h_b, st)

    def _head(self, h, B: int, st: int) -> None:
        """Greedy tokens tok [B] of the rows of h (final RMSNorm, lm_head, argmax)."""
        S = self.spec
        V = self.lm_q.shape[0]
        self._gemm_act(self.lm_q, self.lm_s, h.data_ptr(), _lib.QZ_ACT_RMSNORM,
                       self.norm_w.data_ptr(), self.logits.data_ptr(), max(2, B), V, S.hidden, None,
                       st)
        _lib.check(self.lib.qz_argmax(self.logits.data_ptr(), B, V, self.keys.data_ptr(),
                                      self.tok.data_ptr(), None, 0, st))

    def _plan(self, joins: torch.Tensor, B: int, rows: int) -> qd.KV4Plan:
        return qd.kv4_plan(self.lens[:B], joins, self.table[:B], self.free_pages, self.used,
                           self.page_size, rows, lens_out=self.lens[:B], used_out=self.used)

    # ---------------------------------------------------------------- prompts
    def add(self, prompts: Sequence[Sequence[int]]) -> list[int]:
        """Start requests on non-empty prompts and return their ids; their prompts
        are in the cache afterwards and their first token is decided. Prompts
        share steps of up to max_rows rows; longer ones take several. If a step
        raises, none of the requests is left."""
        prompts = [[int(t) for t in ids] for ids in prompts]
        if not prompts:
            return []
        if any(not ids for ids in prompts):
            raise ValueError("empty prompt: nothing to prefill")
        if any(t < 0 or t >= self.spec.vocab for ids in prompts for t in ids):
            raise ValueError("token id outside the vocabulary")
        if any(len(ids) > self.max_ctx for ids in prompts):
            raise ValueError("prompt does not fit max_ctx")
        if len(self._ids) + len(prompts) > self.max_batch:
            raise ValueError(f"more than max_batch={self.max_batch} requests")
        need = sum(self._pages_of(len(ids)) for ids in prompts)
        if need > self.free:
            raise ValueError(f"prompts need {need} pages, {self.free} are free")
        first, used = len(self._ids), self._used
        try:
            return self._add(prompts)
        except BaseException:
            # the pages that they took are the next of the free list again
            for a in (self._ids, self._len, self._next, self._held):
                del a[first:]
            self._used = used
            self._restore()
            raise

    def _restore(self) -> None:
        """Lengths and cursor on the GPU as the host has them."""
        self.lens[:len(self._len)].copy_(torch.tensor(self._len, dtype=torch.int64))
        self.used.fill_(self._used)

    def _add(self, prompts: list[list[int]]) -> list[int]:
        first = len(self._ids)
        B = first + len(prompts)
        self.lens[first:B].zero_()
        made = list(range(self._serial, self._serial + len(prompts)))
        self._serial += len(prompts)
        self._ids += made
        self._len += [0] * len(prompts)
        self._next += [-1] * len(prompts)
        self._held += [[] for _ in prompts]
        done = [0] * len(prompts)
        with torch.cuda.device(self.dev):
            while any(d < len(ids) for d, ids in zip(done, prompts)):
                room, joins, rows = self.max_rows, [0] * B, []
                for i, ids in enumerate(prompts):
                    n = min(room, len(ids) - done[i])
                    rows += ids[done[i]:done[i] + n]
                    joins[first + i] = n
                    room -= n
                M = max(2, len(rows))          # the GEMMs take two rows or more
                self.ids[:M].copy_(torch.tensor((rows + [0, 0])[:M], dtype=torch.int64))
                plan = self._plan(torch.tensor(joins, dtype=torch.int64).to(self.dev), B, M)
                st = self._stream()
                self._forward(plan, B, M, max(joins), st)
                ends = []                      # requests whose prompt ends with this step
                for i, ids in enumerate(prompts):
                    n = joins[first + i]
                    self._used += self._pages_of(done[i] + n) - self._pages_of(done[i])
                    done[i] += n
                    self._len[first + i] = done[i]
                    if n and done[i] == len(ids):
                        ends.append(i)
                if ends:
                    at = torch.tensor([first + i + 1 for i in ends], device=self.dev)
                    torch.index_select(self.h_a, 0, plan.cu_rows[at] - 1,
                                       out=self.h_last[:len(ends)])
                    self._head(self.h_last, len(ends), st)
                    for i, t in zip(ends, self.tok[:len(ends)].tolist()):
                        self._next[first + i] = t
        return made

    def next_token(self, request: int) -> int:
        """The token that the request's last step decided (not yet in the cache)."""
        return self._next[self._row(request)]

    # ----------------------------------------------------------------- decode
    def _decode_ops(self, B: int) -> None:
        """One step of B requests: tok [B] in, tok [B] out, lengths and pages
        advanced. Every call is a launch on the current stream."""
        M, st = max(2, B), self._stream()
        self.ids[:B].copy_(self.tok[:B])
        plan = self._plan(self.one[:B], B, M)
        self._forward(plan, B, M, 1, st)
        self._head(self.h_a, B, st)

    def _graph(self, B: int) -> torch.cuda.CUDAGraph:
        """The captured step of B requests. The eager step before the capture (it
        settles every launch path) runs on the state and is taken back: lengths,
        tokens and the cursor are restored, and the cache row that it wrote is
        the one that the next step writes again."""
        g = self._graphs.get(B)
        if g is None:
            kept = [t.clone() for t in (self.lens, self.used, self.tok)]
            self._decode_ops(B)
            for t, k in zip((self.lens, self.used, self.tok), kept):
                t.copy_(k)
            side = torch.cuda.Stream(self.dev)
            side.wait_stream(torch.cuda.current_stream(self.dev))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side):
                with torch.cuda.graph(g, stream=side):
                    self._decode_ops(B)
            torch.cuda.current_stream(self.dev).wait_stream(side)
            self._graphs[B] = g
        return g

    def step(self, steps: int = 1, *, graph: bool = True) -> dict[int, list[int]]:
        """Advance every running request by `steps` tokens. Returns request ->
        the tokens it emitted: the one decided before (next_token) first, so the
        first step after add emits the first generated token. What a request
        emitted while generate() ran others comes in front."""
        if not self._ids or steps <= 0:
            return {}
        got = self._advance(steps, graph)
        for row, r in enumerate(self._ids):
            got[r] = self._held[row] + got[r]
            self._held[row] = []
        return got

    def _advance(self, steps: int, graph: bool) -> dict[int, list[int]]:
        """`steps` tokens of every running request."""
        B = len(self._ids)
        if max(self._len) + steps > self.max_ctx:
            raise ValueError("a request would outgrow max_ctx")
        need = sum(self._pages_of(n + steps) - self._pages_of(n) for n in self._len)
        if need > self.free:
            raise ValueError(f"the steps need {need} pages, {self.free} are free")
        try:
            with torch.cuda.device(self.dev):
                self.tok[:B].copy_(torch.tensor(self._next, dtype=torch.int64))
                g = self._graph(B) if graph else None
                out = torch.empty((steps + 1, B), dtype=torch.int64, device=self.dev)
                out[0].copy_(self.tok[:B])
                for i in range(steps):
                    if g is not None:
                        g.replay()
                    else:
                        self._decode_ops(B)
                    out[i + 1].copy_(self.tok[:B])
                got = out.cpu().tolist()
        except BaseException:
            self._restore()          # the requests are where they were before the call
            raise
        self._len = [n + steps for n in self._len]
        self._used += need
        self._next = got[-1]
        return {r: [row[i] for row in got[:-1]] for i, r in enumerate(self._ids)}

    def release(self, request: int) -> None:
        """End a request: its pages are free again and the last running request
        takes its place in the batch."""
        row, last = self._row(request), len(self._ids) - 1
        n = self._pages_of(self._len[row])
        with torch.cuda.device(self.dev):
            if n:
                # pages go back in front of the cursor, the next to be handed out
                self.free_pages[self._used - n:self._used].copy_(self.table[row, :n])
                self.used.sub_(n)
            if row != last:
                self.table[row].copy_(self.table[last])
                self.lens[row:row + 1].copy_(self.lens[last:last + 1])
        self._used -= n
        for a in (self._ids, self._len, self._next, self._held):
            a[row] = a[last]
            a.pop()

    def generate(self, prompts: Sequence[Sequence[int]], steps: int, *, graph: bool = True
                 ) -> list[list[int]]:
        """`steps` greedy tokens after each prompt (prompts of any lengths); the
        requests are released afterwards. Other running requests advance too; the
        next step() returns the tokens that they emit here."""
        if steps <= 0:
            return [[] for _ in prompts]
        ids = self.add(prompts)
        try:
            got = self._advance(steps, graph)
            for row, r in enumerate(self._ids):
                if r not in ids:
                    self._held[row] += got[r]
            return [got[r] for r in ids]
        finally:
            for r in ids:
                self.release(r)
