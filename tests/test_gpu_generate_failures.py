"""generate() leaves every sequence as it was, whatever makes it fail and whenever."""
import numpy as np
import pytest

from test_gpu_batch_step import build, prompt, weights

pytestmark = pytest.mark.gpu


def fails(lstk, m, code, what, prompts, n_new, **kw):
    before = {s: m.seq_len(s) for s in range(12)}
    with pytest.raises(lstk.LstkError) as e:
        m.generate(prompts, n_new, **kw)
    assert e.value.code == code and what in str(e.value), str(e.value)
    assert before == {s: m.seq_len(s) for s in range(12)}


def test_refused_before_the_first_prompt(lstk, dev):
    hp, w = weights("tiny")
    store, m = build(lstk, dev, hp, w, n_batch=4)
    m.decode(1, [1, 2, 3])
    ok = {1: [4, 5], 2: [6]}
    for t in ([1024], [-1], [1, 2 ** 32 + 5], np.array([2 ** 32], np.int64), [1.5], []):
        fails(lstk, m, lstk.E_INVALID, "sequence 2", {1: [4, 5], 2: t}, 3)
    fails(lstk, m, lstk.E_INVALID, "below 0", {1: [4], -2: [5]}, 3)
    fails(lstk, m, lstk.E_INVALID, "sequences", {1: [4], 2 ** 32: [5]}, 3)
    fails(lstk, m, lstk.E_INVALID, "n_sink", ok, 3, window=4, n_sink=-1)
    fails(lstk, m, lstk.E_INVALID, "window", ok, 3, window=2 ** 32 + 1)
    fails(lstk, m, lstk.E_INVALID, "top_k", ok, 3, top_k=np.array([5, 2 ** 32 + 5]))
    fails(lstk, m, lstk.E_INVALID, "setting", ok, 3, top_p=[0.5, 0.5, 0.5])
    got = m.generate(ok, 3, top_k=np.array([5, 7]), temperature=0.5)
    assert [len(t) for t in got.values()] == [3, 3] and m.seq_len(1) == 3 + 2 + 2
    m.close()
    store.close()


def test_cut_back_when_the_cache_is_full(lstk, dev):
    """8 blocks of 32 cells: too few for the second prompt; for both prompts but not for what follows. Afterwards the cells are
    free again, and a call that fits answers like that of a model that never failed."""
    hp, w = weights("tiny")
    store, m = build(lstk, dev, hp, w, n_batch=8, kv_size=256)
    fresh_store, fresh = build(lstk, dev, hp, w, n_batch=8, kv_size=256)
    for x in (m, fresh):
        x.decode(7, prompt(7, 40, 1024))
    long, short = prompt(1, 150, 1024), prompt(2, 60, 1024)
    fails(lstk, m, lstk.E_EXHAUSTED, "full", {0: short, 1: long}, 4)
    fails(lstk, m, lstk.E_EXHAUSTED, "full", {7: [5], 1: long, 0: [3]}, 40)
    assert m.generate({7: [5], 0: short, 1: short}, 6) == fresh.generate({7: [5], 0: short, 1: short}, 6)
    for x in (m, store, fresh, fresh_store):
        x.close()


@pytest.mark.parametrize("n_new", [1, 3])
def test_a_sequence_without_finite_logits(lstk, dev, n_new):
    hp, w = weights("tiny")
    w = dict(w, output_norm=np.full_like(w["output_norm"], np.nan))
    store, m = build(lstk, dev, hp, w, n_batch=4)
    m.decode(4, [1, 2, 3])
    fails(lstk, m, lstk.E_INVALID, "sequence 3 has no finite logit", {3: [1, 2], 4: [3]}, n_new)
    m.close()
    store.close()
