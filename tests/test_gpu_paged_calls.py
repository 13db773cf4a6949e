"""PagedEngine: calls in an order that its other tests do not have."""

import pytest

from tests.test_gpu_paged import _engine, _spec

pytestmark = pytest.mark.gpu

np = pytest.importorskip("numpy")


def _prompts(spec, lengths, seed=8):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, spec.vocab, n).tolist() for n in lengths]


def test_generate_beside_running_requests_loses_no_token():
    """Requests that run while generate() serves others: what they emit meanwhile comes
    with the next step, in order, also after the batch was compacted."""
    spec = _spec()
    eng, _ = _engine(spec)
    prompts = _prompts(spec, (9, 30, 2, 17))
    alone = [eng.generate([p], 16)[0] for p in prompts]
    a, b = eng.add(prompts[:2])
    got = {a: [], b: []}

    def step(n):
        for r, t in eng.step(n).items():
            got[r] += t

    step(2)
    assert eng.generate(prompts[2:], 5) == [t[:5] for t in alone[2:]]
    assert eng.generate([prompts[3]], 4) == [alone[3][:4]]
    assert eng.next_token(a) == alone[0][11]
    step(1)
    assert got == {a: alone[0][:12], b: alone[1][:12]}
    assert eng.generate([prompts[2]], 3) == [alone[2][:3]]
    eng.release(a)                                   # b takes its place in the batch
    del got[a]
    step(1)
    assert got == {b: alone[1][:16]}
    eng.release(b)
    assert eng.free == 64 and eng.running == []


@pytest.mark.parametrize("fails_at", [0, 1, 2])
def test_a_failed_add_leaves_no_requests(monkeypatch, fails_at):
    """An exception in one of add's steps (three of 40 rows here): the engine is as before
    the call, and goes on."""
    spec = _spec()
    eng, _ = _engine(spec)
    prompts = _prompts(spec, (9, 70, 33))
    alone = [eng.generate([p], 8)[0] for p in prompts]
    (a,) = eng.add(prompts[:1])
    assert eng.step(2)[a] == alone[0][:2]
    real, calls = eng._forward, []

    def forward(*args):
        calls.append(args)
        if len(calls) > fails_at:
            raise RuntimeError("planted")
        return real(*args)

    monkeypatch.setattr(eng, "_forward", forward)
    with pytest.raises(RuntimeError, match="planted"):
        eng.add(prompts[1:])
    monkeypatch.undo()
    assert eng.running == [a] and eng.free == 63 and eng.used.item() == 1
    assert eng.step(2)[a] == alone[0][2:4]
    assert eng.generate(prompts[1:], 8) == alone[1:]
    eng.release(a)
    assert eng.free == 64 and sorted(eng.free_pages.tolist()) == list(range(64))


def test_a_failed_step_is_no_step(monkeypatch):
    """An exception after some of a call's steps: lengths and cursor are those before it."""
    spec = _spec()
    eng, _ = _engine(spec)
    prompts = _prompts(spec, (14, 30))
    alone = [eng.generate([p], 12)[0] for p in prompts]
    a, b = eng.add(prompts)
    assert eng.step(1) == {a: alone[0][:1], b: alone[1][:1]}
    real, calls = eng._decode_ops, []

    def ops(B):
        calls.append(B)
        if len(calls) > 3:
            raise KeyboardInterrupt
        return real(B)

    monkeypatch.setattr(eng, "_decode_ops", ops)
    with pytest.raises(KeyboardInterrupt):
        eng.step(5, graph=False)                     # three steps run: both take a new page
    monkeypatch.undo()
    assert eng.length(a) == 15 and eng.lens[:2].tolist() == [15, 31] and eng.free == 64 - 3
    assert eng.step(11) == {a: alone[0][1:], b: alone[1][1:]}
