"""generate() with log probabilities: of every drawn token, as token_logprobs gives them for the step's logits."""
import numpy as np
import pytest

from test_gpu_batch_step import build, prompt, weights

pytestmark = pytest.mark.gpu


def test_of_every_token(lstk, dev):
    """The tokens are those of a run without; the numbers are softmax's over the logits of the same steps run by hand."""
    import torch
    hp, w = weights("tiny")
    V = hp["n_vocab"]
    prompts = {3: prompt(1, 9, V), 0: prompt(2, 30, V), 7: prompt(3, 1, V)}
    how = dict(temperature=[0.9, 0.0, 1.5], top_k=[30, 0, 10], top_p=0.95)
    gen = lambda: torch.Generator(device=dev).manual_seed(11)
    runs = []
    for kw in ({}, dict(logprobs=0), dict(logprobs=4)):
        _, m = build(lstk, dev, hp, w, n_batch=16)
        runs.append(m.generate(prompts, 6, generator=gen(), **how, **kw))
    tokens, said = runs[2]
    assert runs[0] == runs[1][0] == tokens
    _, m = build(lstk, dev, hp, w, n_batch=16)
    logits = torch.empty(3, V, device=dev)
    for i, s in enumerate(prompts):
        m.decode(s, prompts[s], logits=logits[i])
    for step in range(6):
        z = logits.double()
        p = torch.log_softmax(z, 1)
        for i, s in enumerate(prompts):
            d, t = said[s][step], tokens[s][step]
            order = torch.argsort(z[i], descending=True, stable=True)[:4].tolist()
            # (75 + 2 sum p |x - m|) 2^-24 is below 1e-5 here, where no logit that counts is 40 below the largest
            assert abs(d["logprob"] - float(p[i, t])) <= 1e-5 and abs(d["entropy"] + float((p[i].exp() * p[i]).sum())) <= 4e-5
            assert [a for a, _ in d["top"]] == order and all(abs(b - float(p[i, a])) <= 1e-5 for a, b in d["top"])
            assert runs[1][1][s][step] == dict(logprob=d["logprob"], entropy=d["entropy"], top=[])
            if s == 0:
                assert t == order[0]  # the greedy one
        if step < 5:
            m.decode_batch(list(prompts), [tokens[s][step] for s in prompts], logits=logits)
    assert m.generate({}, 3, logprobs=2) == ({}, {}) and m.generate({3: [1]}, 0, logprobs=2) == ({3: []}, {3: []})


@pytest.mark.parametrize("n", [-1, 33, 2 ** 31, "x", 1e300, float("nan")])
def test_refused_before_anything_is_appended(lstk, dev, n):
    hp, w = weights("tiny")
    _, m = build(lstk, dev, hp, w, n_batch=16)
    with pytest.raises(lstk.LstkError) as e:
        m.generate({0: [1, 2]}, 3, logprobs=n)
    assert e.value.code == lstk.E_INVALID and m.seq_len(0) == 0
