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
