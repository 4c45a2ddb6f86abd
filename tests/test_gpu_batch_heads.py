"""Batch steps against the oracle at every head size and at head counts that share a KV head unevenly with 16, and routing by a rule
from hidden rows at a large router. Bars as in test_gpu_batch_step."""
import numpy as np
import pytest

import oracle
from localstack_amd import synth
from test_gpu_batch_step import TINY, build, near, prompt
from test_gpu_select import rule_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_head,n_head_kv,hd,seed", [(4, 2, 128, 1), (8, 1, 128, 2), (4, 4, 256, 3), (20, 1, 64, 4)])
def test_head_sizes(lstk, dev, n_head, n_head_kv, hd, seed):
    """Sequences of 3, 40 and 33 tokens, then batch steps that follow the oracle's own choices: logits of every row."""
    hp = dict(TINY, n_head=n_head, n_head_kv=n_head_kv, head_dim=hd)
    w = synth.qwen3_weights(np.random.default_rng(seed), hp, wtype=8)
    store, model = build(lstk, dev, hp, w)
    refs, feed = {}, {}
    for s, n in enumerate((3, 40, 33)):
        toks = prompt(10 * seed + s, n, hp["n_vocab"])
        refs[s] = oracle.Qwen3(hp, w, 128)
        for i in range(0, n, 16):
            model.decode(s, toks[i:i + 16])
            r = refs[s].decode(toks[i:i + 16])
        feed[s] = int(np.argmax(r))
    for step in range(3):
        order = np.random.default_rng(step).permutation(3)
        got = model.decode_batch(order, [feed[s] for s in order]).cpu().numpy()
        for i, s in enumerate(order):
            ref = refs[s].decode(np.array([feed[s]], np.int32))
            near(got[i], ref, (hd, step, s))
            feed[s] = int(np.argmax(ref))
    model.close()
    store.close()


@pytest.mark.parametrize("T", [1, 200])
def test_route_by_over_128_experts(lstk, dev, T):
    """Weights against the rule on the router's logits in 64 bits, whose fp32 sums are off by at most h 2^-24 sum |x w|; ids wherever the
    neighbouring choice values lie further apart than that moves them."""
    import torch
    h, f, E, k = 512, 512, 128, 8
    rng = np.random.default_rng(T)
    types = (8, 8, 8)
    layer = (types, synth.experts(rng, 8, E, f, h), synth.experts(rng, 8, E, f, h), synth.experts(rng, 8, E, h, f))
    store = lstk.ExpertStore(1, h, f, E, k, 256, [layer])
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    gate, x = synth.router_f16(rng, E, h), synth.activations(rng, T, h)
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    ids, wts = torch.zeros(T, k, dtype=torch.int32, device=dev), torch.zeros(T, k, device=dev)
    rule = dict(score="sigmoid", n_group=8, n_group_used=4, group_top=2, scale=2.5)
    store.route_by(0, lstk.RouterRule(**rule), d(x), d(gate), lstk.TYPE_F16, ids, wts, bias=d(bias))
    a, b = x.astype(np.float16).astype(np.float64), gate.view(np.float16).reshape(E, h).astype(np.float64)
    lg = (a @ b.T).astype(np.float32)
    off = 0.25 * h * 2.0 ** -24 * (np.abs(a) @ np.abs(b).T).max() + 2.0 ** -23  # of a score: a sigmoid's slope is at most 1 / 4
    want, ww = rule_of(lg, k, bias=bias, **rule)
    c = 1 / (1 + np.exp(-lg.astype(np.float64))) + bias
    groups = -np.sort(-(-np.sort(-c.reshape(T, 8, 16), axis=2)[:, :, :2]).sum(2), axis=1)
    kept = rule_of(lg, k + 1, bias=bias, **rule)[0]
    gaps = -np.diff(np.take_along_axis(c, kept, 1), axis=1)
    clear = (gaps > 2 * off).all(1) & (groups[:, 3] - groups[:, 4] > 4 * off)
    assert clear.mean() > 0.9
    np.testing.assert_array_equal(ids.cpu().numpy()[clear], want[clear])
    s = np.take_along_axis(c - bias, want, 1).sum(1, keepdims=True)
    assert (np.abs(wts.cpu().numpy() - ww)[clear] <= (2.5 * off * (1 + k) / s + 2.0 ** -23 * ww)[clear]).all()
    out, resid = torch.zeros(T, h, device=dev), d(synth.activations(rng, T, h))
    store.ffn(0, d(x), ids, wts, resid, out)
    store.check()
    assert torch.isfinite(out).all()
    store.close()
