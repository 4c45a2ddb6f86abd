"""The two halves of a step belong together: forward() does not run on what prepare_batch() left."""
import pytest

from test_gpu_batch_step import LOGITS_TOL, build, prompt, weights

pytestmark = pytest.mark.gpu


def test_forward_after_a_batch_step(lstk, dev):
    import torch
    hp, w = weights("tiny")
    (store, m), (ref_store, ref) = (build(lstk, dev, hp, w, n_batch=4) for _ in range(2))
    for x in (m, ref):
        for s in range(2):
            x.decode(s, prompt(s, 20, 1024))
    for step in (lambda: m.prepare_batch([0, 1], [5, 6]), lambda: m.forward_batch(2, 64)):
        step()
        with pytest.raises(lstk.LstkError) as e:
            m.forward(0, 1, 256)
        assert e.value.code == lstk.E_INVALID and "batch" in str(e.value)
    ref.decode_batch([0, 1], [5, 6])
    # prepared as its own step it runs
    n = m.prepare(0, [7])
    assert torch.equal(m.forward(0, 1, n), ref.decode(0, [7]))
    # a capture that follows a batch step records the step, and its replays run on what prepare() left
    m.decode_batch([1, 0], [8, 9])
    ref.decode_batch([1, 0], [8, 9])
    logits = torch.empty(1024, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.forward(0, 1, n, logits=logits)
    for t in (11, 12, 13):
        assert m.prepare(0, [t]) == n
        g.replay()
        want = ref.decode(0, [t])
        assert float((logits - want).abs().max()) <= LOGITS_TOL  # (a capture's attention is cut up differently)
        m.decode_batch([1], [t])
        ref.decode_batch([1], [t])
    for x in (m, store, ref, ref_store):
        x.close()
