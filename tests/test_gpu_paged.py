"""The paged 4-bit engine against a plain 64-bit decoder that quantises its K and V
rows by the same definition (tests/_kv4.py), and its bookkeeping.

A K or V value that lies within fp32 rounding of the middle between two codes may
get the neighbouring code here and there; one such code moves a score by a
fifteenth of a row's range times one query value, so logits are compared with
1 % of their spread and tokens where the two best differ by more than that.
"""

import pytest

from tests import _kv4 as P

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
np = pytest.importorskip("numpy")


def _spec(arch="Qwen3ForCausalLM", hd=64, nq=4, nkv=2, **kw):
    from quartz_b200.model import ModelSpec
    return ModelSpec(**dict(dict(arch=arch, hidden=256, layers=2, n_heads=nq, n_kv=nkv, head_dim=hd,
                                 inter=512, vocab=700, rope_theta=1e4, tie=True), **kw))


def _engine(spec, **kw):
    from quartz_b200.model import norm_weights, random_int8_weights
    from quartz_b200.paged import PagedEngine
    w = {n: (q, s) for n, q, s in random_int8_weights(spec, seed=3, std=0.08)}
    kw = dict(dict(pages=64, max_ctx=256, max_batch=6, page_size=16, max_rows=40), **kw)
    return PagedEngine(spec, w, norm_weights(spec), **kw), w


class Plain:
    """One request, token by token, fp64 with 4-bit K and V."""

    def __init__(self, spec, weights):
        from quartz_b200.model import rope_inv_freq
        self.S = spec
        self.w = {n: torch.from_numpy(q).double() * torch.from_numpy(s).double() for n, (q, s) in weights.items()}
        self.inv = torch.from_numpy(rope_inv_freq(spec))
        self.k = [[] for _ in range(spec.layers)]
        self.v = [[] for _ in range(spec.layers)]

    def _norm(self, x):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + self.S.eps)

    def _rope(self, x, pos):
        ang = (torch.tensor(float(pos), dtype=torch.float32) * self.inv).double()
        c, s = torch.cos(ang), torch.sin(ang)
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    def feed(self, tok):
        S, w = self.S, self.w
        h = w["model.embed_tokens"][tok]
        for i in range(S.layers):
            p = f"model.layers.{i}."
            pos = len(self.k[i])
            x = self._norm(h)
            q = (w[p + "self_attn.q_proj"] @ x).view(S.n_heads, -1)
            k = (w[p + "self_attn.k_proj"] @ x).view(S.n_kv, -1)
            v = (w[p + "self_attn.v_proj"] @ x).view(S.n_kv, -1)
            if S.qk_norm:
                q, k = self._norm(q), self._norm(k)
            q, k = self._rope(q, pos), self._rope(k, pos)
            self.k[i].append(P.values(k.float()))
            self.v[i].append(P.values(v.float()))
            kk, vv = (torch.stack(t).transpose(0, 1).repeat_interleave(S.n_heads // S.n_kv, 0)
                      for t in (self.k[i], self.v[i]))
            a = torch.softmax((kk * q[:, None]).sum(-1) * S.head_dim ** -0.5, -1)
            h = h + w[p + "self_attn.o_proj"] @ (a[..., None] * vv).sum(1).flatten()
            x = self._norm(h)
            g, u = w[p + "mlp.gate_proj"] @ x, w[p + "mlp.up_proj"] @ x
            h = h + w[p + "mlp.down_proj"] @ (g / (1 + torch.exp(-g)) * u)
        return w["model.embed_tokens"] @ self._norm(h)


def _close(logits, ref):
    spread = (ref.max() - ref.min()).item()
    assert (logits.double().cpu() - ref).abs().max().item() < 0.01 * spread
    top = ref.topk(2).values
    return (top[0] - top[1]).item() > 0.02 * spread


@pytest.mark.parametrize("arch,hd,nq,nkv,page", [("Qwen3ForCausalLM", 64, 4, 2, 16),
                                                 ("LlamaForCausalLM", 64, 8, 1, 32),
                                                 ("Qwen3ForCausalLM", 128, 6, 2, 64)])
def test_engine_against_the_plain_decoder(arch, hd, nq, nkv, page):
    spec = _spec(arch, hd, nq, nkv)
    eng, w = _engine(spec, page_size=page)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, spec.vocab, n).tolist() for n in (1, 17, 53, 5)]   # 76 rows: two steps
    plain = [Plain(spec, w) for _ in prompts]
    refs = []
    for pl, ids in zip(plain, prompts):
        for t in ids:
            ref = pl.feed(t)
        refs.append(ref)
    reqs = eng.add(prompts)
    checked = 0
    for r, ref in zip(reqs, refs):
        spread = (ref.max() - ref.min()).item()
        top = ref.topk(2)
        if (top.values[0] - top.values[1]).item() > 0.02 * spread:
            assert eng.next_token(r) == top.indices[0].item()
            checked += 1
    # the cache holds the rows of the definition, up to codes on a border
    for r, pl in zip(reqs, plain):
        for layer in range(spec.layers):
            k, v = eng.kv(r, layer)
            for got, want in ((k, pl.k[layer]), (v, pl.v[layer])):
                want = torch.stack(want)
                assert got.shape == want.shape
                off = (got.double().cpu() - want).abs() > 0.02 * want.abs().max()
                assert off.double().mean().item() < 0.02
    # the plain decoders follow the engine's tokens
    for _ in range(12):
        toks = [eng.next_token(r) for r in reqs]
        out = eng.step(1)
        assert [out[r] for r in reqs] == [[t] for t in toks]
        for i, (r, pl) in enumerate(zip(reqs, plain)):
            ref = pl.feed(toks[i])
            if _close(eng.logits[eng.running.index(r)], ref):
                assert eng.next_token(r) == ref.argmax().item()
                checked += 1
    assert checked > 20
    from quartz_b200 import device as qd
    qd.check_status()


def test_batches_graphs_and_order_do_not_change_tokens():
    spec = _spec()
    eng, _ = _engine(spec)
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, spec.vocab, n).tolist() for n in (9, 30, 2, 61)]
    together = eng.generate(prompts, 20)
    assert eng.free == 64 and eng.used.item() == 0 and eng.running == []
    assert eng.generate(prompts, 20, graph=False) == together
    alone = [eng.generate([p], 20)[0] for p in prompts]
    assert alone == together
    # requests that start and end while others run
    a, b = eng.add(prompts[:2])
    got = {a: [], b: []}
    for r, t in eng.step(5).items():
        got[r] += t
    (c,) = eng.add([prompts[2]])
    got[c] = []
    for r, t in eng.step(7).items():
        got[r] += t
    eng.release(a)
    (d,) = eng.add([prompts[3]])
    got[d] = []
    for r, t in eng.step(8).items():
        got[r] += t
    for r, i in ((a, 0), (b, 1), (c, 2), (d, 3)):
        assert got[r] == together[i][:len(got[r])], i
    for r in (b, c, d):
        eng.release(r)
    assert eng.free == 64 and eng.used.item() == 0
    assert sorted(eng.free_pages.tolist()) == list(range(64))     # every page once


def test_engine_refuses():
    spec = _spec()
    eng, _ = _engine(spec, pages=8, max_batch=2, max_ctx=100)
    with pytest.raises(ValueError, match="empty prompt"):
        eng.add([[]])
    with pytest.raises(ValueError, match="vocabulary"):
        eng.add([[spec.vocab]])
    with pytest.raises(ValueError, match="max_ctx"):
        eng.add([[1] * 101])
    with pytest.raises(ValueError, match="max_batch"):
        eng.add([[1], [2], [3]])
    with pytest.raises(ValueError, match="pages"):
        eng.add([[1] * 70, [2] * 70])
    assert eng.running == [] and eng.free == 8
    (r,) = eng.add([[1] * 90])
    with pytest.raises(ValueError, match="max_ctx"):
        eng.step(11)
    (s,) = eng.add([[2] * 30])
    with pytest.raises(ValueError, match="pages"):
        eng.step(7)
    eng.release(r)
    assert eng.length(s) == 30 and len(eng.step(7)[s]) == 7
    with pytest.raises(KeyError):
        eng.release(r)
    assert eng.add([]) == [] and eng.step(0) == {}
    from quartz_b200.paged import PagedEngine
    with pytest.raises(ValueError, match="page_size"):
        PagedEngine(spec, {}, {}, pages=4, max_ctx=10, page_size=48)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_and_append_in_one_launch(hd, norm):
    """qk_rope_kv4 against qk_rope into an fp32 cache followed by kv4_append."""
    from quartz_b200 import device as qd
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(hd)
    nq, nkv, M, page = 6, 2, 37, 16
    qkv = torch.randn(M, (nq + 2 * nkv) * hd, generator=g, device=dev)
    inv = torch.rand(hd // 2, generator=g, device=dev)
    qn, kn = (torch.rand(hd, generator=g, device=dev) + 0.5 for _ in range(2)) if norm else (None, None)
    pool = qd.kv4_pool(6, nkv, hd, page, dev)
    slots = torch.randperm(6 * page, generator=g, device=dev)[:M].clone()
    pos0 = 11
    positions = torch.arange(M, device=dev) + pos0
    q = qd.qk_rope_kv4(qkv, inv, positions, pool, slots, nq, qn, kn, 1e-6)
    kc, vc = (torch.zeros(nkv, pos0 + M, hd, device=dev) for _ in range(2))
    q_ref = qd.qk_rope(qkv, inv, kc, vc, nq, pos0=pos0, q_norm=qn, k_norm=kn, eps=1e-6)
    assert (q.view_as(q_ref) - q_ref).abs().max() < 1e-5
    k, v = kc[:, pos0:].transpose(0, 1).contiguous(), vc[:, pos0:].transpose(0, 1).contiguous()
    gk, gv = qd.kv4_gather(pool, slots, hd)
    assert torch.equal(gv, P.values(v).float())             # v is stored as it is
    off = (gk.double() - P.values(k)).abs() > 1e-4
    assert off.double().mean() < 0.002                      # codes on a border
    # padding rows: nothing stored, q written
    before = pool.clone()
    slots.fill_(-1)
    positions.fill_(-1)
    qd.qk_rope_kv4(qkv, inv, positions, pool, slots, nq, qn, kn, 1e-6, q_out=q)
    assert torch.equal(pool, before) and torch.isfinite(q).all()
