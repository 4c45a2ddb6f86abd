"""Routing by a rule (lstk_moe_select, lstk_moe_route_by) against the rule in 64 bits with numpy.

Ids have to be equal: choice values are 64-bit on both sides and the seeds' neighbours lie further apart than their
roundings (asserted). A weight is a 64-bit quotient rounded once to fp32: 2^-24 relative, and 2^-44 for the 64-bit steps."""
import numpy as np
import pytest

from localstack_amd import synth

pytestmark = pytest.mark.gpu

FMAX = np.finfo(np.float32).max


def rule_of(x, k, score="softmax", n_group=1, n_group_used=None, group_top=1, renorm=True, scale=1.0, bias=None):
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, FMAX)).astype(np.float64)
    T, E = x.shape
    used = n_group if n_group_used is None else n_group_used
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        if score == "softmax":
            top = x.max(1, keepdims=True)
            p = np.exp(x - np.where(np.isinf(top), 0, top))
            t = p.sum(1, keepdims=True)
            p = np.where(t > 0, p / np.where(t > 0, t, 1), 0)
        else:
            p = 1 / (1 + np.exp(-x))
        c = p if bias is None else p + bias.astype(np.float64)
    c = np.where(np.isnan(c), -np.inf, c)
    out = np.ones((T, E), bool)
    if used < n_group:
        per = E // n_group
        s = -np.sort(-c.reshape(T, n_group, per), axis=2)
        with np.errstate(invalid="ignore"):
            v = s[:, :, 0] if group_top == 1 else s[:, :, 0] + s[:, :, 1]
        v = np.where(np.isnan(v), -np.inf, v)
        keep = np.argsort(-v, axis=1, kind="stable")[:, :used]
        out = np.zeros((T, n_group), bool)
        np.put_along_axis(out, keep, True, 1)
        out = np.repeat(out, per, axis=1)
    ids = np.zeros((T, k), np.int64)
    for t in range(T):
        e = np.flatnonzero(out[t])
        ids[t] = e[np.argsort(-c[t, e], kind="stable")[:k]]
    w = np.take_along_axis(p, ids, 1)
    if renorm:
        w = w / np.maximum(w.sum(1, keepdims=True), 2.0 ** -14)
    return ids, w * np.float64(np.float32(scale))


def check(lstk, dev, x, k, bias=None, xd=None, **rule):
    import torch
    xd = torch.from_numpy(x).to(dev) if xd is None else xd
    b = None if bias is None else torch.from_numpy(bias).to(dev)
    ids, w = lstk.moe_select(xd, k, lstk.RouterRule(**rule), bias=b)
    want, ww = rule_of(x, k, bias=bias, **rule)
    np.testing.assert_array_equal(ids.cpu().numpy(), want)
    got = w.cpu().numpy().astype(np.float64)
    assert (np.abs(got - ww) <= np.abs(ww) * (2.0 ** -24 + 2.0 ** -44) + 2.0 ** -149).all()
    return ids, w


def logits(rng, T, E):
    return (1.5 * rng.standard_normal((T, E)) + rng.standard_normal((1, E))).astype(np.float32)


@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (2, 2), (8, 2), (60, 4), (63, 7), (64, 8), (65, 8), (96, 6), (128, 8), (160, 6), (200, 64), (256, 8),
                                 (256, 64), (64, 64)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_sizes(lstk, dev, E, k, score):
    rng = np.random.default_rng(E * 100 + k)
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    for T in (1, 3, 4, 5, 257):
        x = logits(rng, T, E)
        check(lstk, dev, x, k, score=score)
        check(lstk, dev, x, k, bias=bias, score=score, renorm=False, scale=2.5)


@pytest.mark.parametrize("E,k,G,used,top", [(256, 8, 8, 4, 2), (256, 8, 8, 1, 1), (160, 6, 8, 3, 1), (64, 6, 4, 2, 2), (128, 8, 16, 5, 2), (6, 2, 3, 1, 2),
                                            (8, 4, 8, 4, 1), (256, 4, 256, 4, 1), (256, 64, 2, 1, 2), (60, 5, 5, 2, 1), (128, 8, 128, 100, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups(lstk, dev, E, k, G, used, top, score):
    rng = np.random.default_rng(E + 7 * G + used)
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    for T in (1, 130):
        x = logits(rng, T, E)
        for b in (None, bias):
            check(lstk, dev, x, k, bias=b, score=score, n_group=G, n_group_used=used, group_top=top, scale=1.5)


def test_many_tokens(lstk, dev):
    rng = np.random.default_rng(2)
    check(lstk, dev, logits(rng, 30001, 128), 8)
    check(lstk, dev, logits(rng, 20000, 256), 8, bias=(0.1 * rng.standard_normal(256)).astype(np.float32), score="sigmoid", n_group=8,
          n_group_used=4, group_top=2, scale=2.5)


def test_ties_go_to_the_lower_id(lstk, dev):
    x = np.zeros((3, 128), np.float32)
    x[1, ::2] = 1.0
    x[2] = np.repeat(np.arange(16), 8)
    for score in ("softmax", "sigmoid"):
        check(lstk, dev, x, 8, score=score)
        check(lstk, dev, x, 8, score=score, n_group=8, n_group_used=3, group_top=2)
        check(lstk, dev, x, 8, score=score, bias=np.ones(128, np.float32))


def test_special_values(lstk, dev):
    """-inf (an expert switched off), NaN (as -inf), +inf, rows of nothing but those, scores that under- and overflow."""
    inf, nan = np.inf, np.nan
    x = np.array([[0, 1, 2, 3, 4, 5, 6, 7], [-inf] * 8, [nan] * 8, [-inf, -inf, 3, -inf, nan, 1, -inf, -inf], [inf, 0, inf, -inf, 1, 2, 3, 4],
                  [FMAX, FMAX, -FMAX, 0, 1, 2, 3, 4], [800, -800, 0, 1, 90, -90, 40, -40], [-1000, -1001, -1002, -999, -998, -2000, -1000, -1000],
                  [1e-30, 0, -1e-30, -0.0, 1e-38, 0, 0, 0]], np.float32)
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            check(lstk, dev, x, 3, score=score, renorm=renorm)
            check(lstk, dev, x, 3, score=score, renorm=renorm, n_group=4, n_group_used=2, group_top=2)
            for b in ([0, -inf, 0, -inf, 0, 0, 0, 0], [nan, 0, 0, 0, 0, 0, 0, inf], [-inf] * 8, [1e30, 0, 0, 0, -1e30, 0, 0, 0]):
                check(lstk, dev, x, 3, bias=np.array(b, np.float32), score=score, renorm=renorm)
                check(lstk, dev, x, 2, bias=np.array(b, np.float32), score=score, renorm=renorm, n_group=4, n_group_used=1, group_top=2)


def test_strided_rows(lstk, dev):
    import torch
    rng = np.random.default_rng(3)
    x = logits(rng, 50, 128)
    for off, ld in ((0, 200), (1, 131), (3, 160)):
        big = torch.full((50, off + ld), 99.0, device=dev)
        v = big[:, off:off + 128]
        v.copy_(torch.from_numpy(x))
        check(lstk, dev, x, 8, xd=v)


def test_rows_behind_stay_and_capture(lstk, dev):
    import torch
    rng = np.random.default_rng(4)
    x = torch.from_numpy(logits(rng, 70, 256)).to(dev)
    ids, w = torch.full((80, 8), -7, dtype=torch.int32, device=dev), torch.full((80, 8), -7.0, device=dev)
    rule = lstk.RouterRule("sigmoid", 8, 4, 2, True, 2.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    lstk.moe_select(x, 8, rule, ids=ids[:70], weights=w[:70], stream=side)
    side.synchronize()
    assert (ids[70:] == -7).all() and (w[70:] == -7.0).all() and (ids[:70] >= 0).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lstk.moe_select(x, 8, rule, ids=ids[:70], weights=w[:70])
    for _ in range(4):
        x.copy_(x.roll(1, 1))
        g.replay()
        a, b = lstk.moe_select(x, 8, rule)
        assert torch.equal(a, ids[:70]) and torch.equal(b, w[:70])


@pytest.mark.parametrize("T", [1, 7, 40])
def test_route_by_matches_route_and_feeds_the_experts(lstk, dev, T):
    """On a pool: softmax + top-k + renormalise gives lstk_moe_route's ids, and its weights to fp32 rounding; a sigmoid rule with
    bias and groups gives the rule's result on the router's own logits, and its ids and weights run through ffn()."""
    import torch
    h, f, E, k = 256, 512, 16, 4
    rng = np.random.default_rng(50 + T)
    types = (8, 8, 8)
    store = lstk.ExpertStore(1, h, f, E, k, 64, [(types, synth.experts(rng, 8, E, f, h), synth.experts(rng, 8, E, f, h),
                                                  synth.experts(rng, 8, E, h, f))])
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    gate = synth.router_f16(rng, E, h)
    x = synth.activations(rng, T, h)
    xd, gd = d(x), d(gate)
    new = lambda: (torch.full((T, k), -1, dtype=torch.int32, device=dev), torch.zeros(T, k, device=dev))
    (i0, w0), (i1, w1), (i2, w2) = new(), new(), new()
    store.route(0, xd, gd, lstk.TYPE_F16, i0, w0)
    store.route_by(0, lstk.RouterRule(), xd, gd, lstk.TYPE_F16, i1, w1)
    assert torch.equal(i0, i1)
    assert float((w0 - w1).abs().max()) <= 1e-6
    bias = (0.2 * rng.standard_normal(E)).astype(np.float32)
    rule = dict(score="sigmoid", n_group=4, n_group_used=2, group_top=2, scale=2.0)
    store.route_by(0, lstk.RouterRule(**rule), xd, gd, lstk.TYPE_F16, i2, w2, bias=d(bias))
    lg = (x.astype(np.float16).astype(np.float64) @ gate.view(np.float16).reshape(E, h).astype(np.float64).T).astype(np.float32)
    want, ww = rule_of(lg, k, bias=bias, **rule)
    np.testing.assert_array_equal(i2.cpu().numpy(), want)
    assert np.abs(w2.cpu().numpy() - ww).max() <= 1e-5  # the logits' own fp32 summation order
    out = torch.zeros(T, h, device=dev)
    resid = d(synth.activations(rng, T, h))
    store.ffn(0, xd, i2, w2, resid, out)
    store.check()
    a = out.clone()
    # the same experts in another order, weights with them: the same sum
    perm = [2, 0, 3, 1]
    store.ffn(0, xd, i2[:, perm].contiguous(), w2[:, perm].contiguous(), resid, out)
    store.check()
    assert float((a - out).abs().max()) <= 1e-4 * float((a - resid).abs().max() + 1)
    for bad in (dict(score="sigmoid", n_group=3), dict(n_group=4, n_group_used=1, group_top=2), dict(n_group=16, group_top=2)):
        r = lstk.RouterRule(**bad)
        if bad.get("n_group_used") == 1:
            store.route_by(0, r, xd, gd, lstk.TYPE_F16, i2, w2)  # one group of four holds the four experts
            continue
        with pytest.raises(lstk.LstkError) as e:
            store.route_by(0, r, xd, gd, lstk.TYPE_F16, i2, w2)
        assert e.value.code == lstk.E_INVALID
    store.close()


def test_refusals_of_tensors(lstk, dev):
    import torch
    x = torch.zeros(3, 16, device=dev)
    R = lstk.RouterRule
    lstk.moe_select(x, 2, R())
    for args, kw in (((x.half(), 2, R()), {}), ((x.cpu(), 2, R()), {}), ((x[0], 2, R()), {}), ((x.t(), 2, R()), {}), ((x, 0, R()), {}),
                     ((x, 17, R()), {}), ((x, 2, R(n_group=3)), {}), ((x, 2, R(n_group=0)), {}), ((x, 2, R(n_group=4, n_group_used=5)), {}),
                     ((x, 5, R(n_group=4, n_group_used=1)), {}), ((x, 2, R(group_top=3)), {}), ((x, 2, R(n_group=16, group_top=2)), {}),
                     ((x, 2, R(scale=float("nan"))), {}), ((torch.zeros(2, 257, device=dev), 2, R()), {}),
                     ((torch.zeros(2, 0, device=dev), 1, R()), {}), ((x, 2, R()), dict(bias=torch.zeros(15, device=dev))),
                     ((x, 2, R()), dict(bias=torch.zeros(16, device=dev).double())), ((x, 2, R()), dict(ids=torch.zeros(3, 2, device=dev))),
                     ((x, 2, R()), dict(weights=torch.zeros(2, 2, device=dev)))):
        with pytest.raises(lstk.LstkError) as e:
            lstk.moe_select(*args, **kw)
        assert e.value.code == lstk.E_INVALID
    a, b = lstk.moe_select(x[:0], 2, R())
    assert a.shape == b.shape == (0, 2)
