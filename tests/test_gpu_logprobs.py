"""Log probabilities of given tokens, entropy and the largest values (lstk_token_logprobs) against numpy in 64 bits.

Tolerance, from the kernel's arithmetic (u = 2^-24): a term e^(x - m) is off by (2 + 2 |x - m|) u relative (the difference's rounding, its
product with log2 e and that constant's own rounding; the exponential), sums of a thread's up to 64 values and of its wavefront add (64 + 8) u.
So with D = sum p |x - m|: ln l is off by (75 + 2 D) u, a log probability by that and its own rounding, the entropy by
(75 + 2 D) u (1 + D) + 2 u sum p |x - m|^2 and its rounding.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def expect(x, tokens, n):
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
    V = x.shape[1]
    m = x.max(1)
    some = m > -np.inf
    z = x - np.where(some, m, 0.0)[:, None]
    w = np.exp(z)
    l = np.where(some, w.sum(1), 1.0)
    zf = np.where(w > 0, z, 0.0)
    p = w / l[:, None]
    lse = np.log(l)
    D = (p * np.abs(zf)).sum(1)
    entropy = np.where(some, lse + D, 0.0)
    tol_l = (75 + 2 * D) * U
    tol_e = tol_l * (1 + D) + 2 * U * (p * zf * zf).sum(1) + U * np.abs(entropy)
    inside = (tokens >= 0) & (tokens < V)
    of = np.where(inside, z[np.arange(len(x)), np.where(inside, tokens, 0)] - lse, -np.inf)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :n]
    at = np.take_along_axis(z, ids, 1) - lse[:, None]
    ids = np.where(at > -np.inf, ids, -1)
    if ids.shape[1] < n:
        pad = n - ids.shape[1]
        ids, at = np.pad(ids, ((0, 0), (0, pad)), constant_values=-1), np.pad(at, ((0, 0), (0, pad)), constant_values=-np.inf)
    return of, entropy, ids, at, tol_l, tol_e


def close(got, want, tol):
    got, tol = got.astype(np.float64), np.broadcast_to(tol, want.shape)
    # two logits at the ends of fp32 are up to 6.8e38 apart, and the nearest fp32 number to -6.8e38 is -inf
    with np.errstate(over="ignore"):
        want = np.where(np.isinf(want.astype(np.float32)), want.astype(np.float32), want)
    far = np.isinf(want)
    assert np.array_equal(got[far], want[far])
    err = np.abs(got[~far] - want[~far])
    assert (err <= tol[~far] + U * np.abs(want[~far])).all(), float((err - tol[~far]).max())


def check(lstk, dev, x, tokens, n, **kw):
    import torch
    xd = torch.from_numpy(x).to(dev) if isinstance(x, np.ndarray) else x
    r = lstk.token_logprobs(xd, torch.tensor(tokens, dtype=torch.int32, device=dev), n_top=n, **kw)
    of, entropy, ids, at, tol_l, tol_e = expect(xd.cpu().numpy(), np.asarray(tokens, np.int64), n)
    g = [t.cpu().numpy() for t in r]
    assert np.array_equal(g[2], ids)
    close(g[0], of, tol_l)
    close(g[1], entropy, tol_e)
    close(g[3], at, tol_l[:, None])
    return r


def logits(rng, n, V, spread=2.2, ahead=8.0):
    x = spread * rng.standard_normal((n, V))
    k = min(V, 40)
    for r in range(n):
        at = rng.choice(V, k, replace=False)
        x[r, at] += ahead * rng.random(k)
    return x.astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 3, 5, 31, 64, 1000, 1023, 1024, 4093, 16380, 16384, 16387, 50259, 151936, 300001])
@pytest.mark.parametrize("n", [0, 1, 20, 32])
def test_vocabularies(lstk, dev, V, n):
    rng = np.random.default_rng(V + n)
    rows = 5
    check(lstk, dev, logits(rng, rows, V), rng.integers(0, V, rows), n)


@pytest.mark.parametrize("rows,V", [(1, 151936), (64, 151936), (300, 5001), (700, 129), (130, 40003)])
def test_rows(lstk, dev, rows, V):
    rng = np.random.default_rng(rows)
    check(lstk, dev, logits(rng, rows, V), rng.integers(0, V, rows), 8)


def test_largest_vocabulary(lstk, dev):
    import torch
    V = 2 ** 20 - 16
    rng = np.random.default_rng(1)
    x = logits(rng, 2, V)
    wide = torch.from_numpy(np.pad(x, ((0, 0), (3, 2)))).to(dev)  # rows out of line
    check(lstk, dev, wide[:, 3:3 + V], [V - 1, 0], 32)


def test_strided_rows(lstk, dev):
    """Rows inside wider ones, at every place of a 16-byte unit; what lies beside them (NaN) is not looked at."""
    import torch
    rng = np.random.default_rng(2)
    for V in (7, 1001, 20001):
        for at in range(4):
            wide = torch.full((6, V + 9), float("nan"), device=dev)
            wide[:, at:at + V] = torch.from_numpy(logits(rng, 6, V)).to(dev)
            check(lstk, dev, wide[:, at:at + V], rng.integers(0, V, 6), 5)


def test_a_certain_token(lstk, dev):
    """One value far above the others: its log probability is 0 or a little below, the others' are the distances."""
    rng = np.random.default_rng(3)
    x = logits(rng, 4, 151936)
    for r, d in enumerate((12.0, 25.0, 90.0, 3000.0)):
        x[r, 1000 * r + 7] = x[r].max() + d
    check(lstk, dev, x, [7, 1007, 2007, 3007], 5)
    check(lstk, dev, x, [8, 9, 10, 11], 5)


def test_equal_values(lstk, dev):
    """Ties go to the lowest ids, whole rows of equal values among them; -0 and 0 are equal."""
    for V in (40, 3000, 50000):
        x = np.zeros((4, V), np.float32)
        x[1] = -np.float32(3.5)
        x[2, ::2] = -0.0
        x[3, ::3] = 1.0
        check(lstk, dev, x, [0, V - 1, V // 2, 3], 32)
    x = np.round(np.random.default_rng(4).standard_normal((6, 20000))).astype(np.float32)
    check(lstk, dev, x, [0, 1, 2, 3, 4, 5], 20)


def test_rows_of_which_little_may_come(lstk, dev):
    """-inf, NaN and +inf: only a few values above -inf, none at all, and values at the ends of fp32."""
    rng = np.random.default_rng(5)
    for V in (50, 5000, 60000):
        x = logits(rng, 9, V)
        x[0, rng.random(V) < 0.9] = -np.inf
        x[1, 3:] = -np.inf
        x[2] = -np.inf
        x[3] = np.nan
        x[4, 5:20] = np.nan
        x[5, V - 2] = np.inf
        x[6, [1, V - 1]] = np.inf
        x[7] = -np.finfo(np.float32).max
        x[8] = np.where(np.arange(V) % 2 == 0, np.finfo(np.float32).max, -np.finfo(np.float32).max)
        check(lstk, dev, x, [0, 1, 2, 3, 6, V - 2, 1, 0, 1], 20)
        check(lstk, dev, x, [0, V - 1, V - 2, 3, 5, 0, 0, 0, 0], 0)


def test_tokens_outside_the_vocabulary(lstk, dev):
    rng = np.random.default_rng(6)
    check(lstk, dev, logits(rng, 5, 500), [-1, 500, 2 ** 31 - 1, -2 ** 31, 499], 3)


def test_buffers_streams_and_capture(lstk, dev):
    import torch
    rng = np.random.default_rng(7)
    x = torch.from_numpy(logits(rng, 8, 50000)).to(dev)
    tok = torch.arange(8, dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = lstk.token_logprobs(x, tok, n_top=4, stream=side)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, lstk.token_logprobs(x, tok, n_top=4)))
    need = lstk.token_logprobs_work_bytes(8, 50000, 4)
    work = torch.full((need + 64,), 9, dtype=torch.uint8, device=dev)
    big = dict(logprobs=torch.full((10,), 7.0, device=dev), entropy=torch.full((10,), 7.0, device=dev),
               top_ids=torch.full((10, 4), 7, dtype=torch.int32, device=dev), top_logprobs=torch.full((10, 4), 7.0, device=dev))
    lstk.token_logprobs(x, tok, n_top=4, work=work[:need], **{k: v[:8] for k, v in big.items()})
    for p, (_, v) in zip(a, big.items()):
        assert torch.equal(v[:8], p) and (v[8:] == 7).all()
    assert (work[need:] == 9).all()
    graphs = []
    for n in (0, 6):
        w = torch.empty(lstk.token_logprobs_work_bytes(8, 50000, n), dtype=torch.uint8, device=dev)
        o = (torch.zeros(8, device=dev), torch.zeros(8, device=dev), torch.zeros(8, n, dtype=torch.int32, device=dev), torch.zeros(8, n, device=dev))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lstk.token_logprobs(x, tok, n, *o, work=w)
        graphs.append((n, g, o, w))
    for step in range(4):
        x.copy_(torch.from_numpy(logits(rng, 8, 50000)))
        tok.add_(100 * step)
        for _, g, _, _ in graphs:
            g.replay()
        for n, _, o, _ in graphs:
            assert all(torch.equal(p, q) for p, q in zip(o, lstk.token_logprobs(x, tok, n_top=n))), (step, n)


def test_refusals_of_tensors(lstk, dev):
    import torch
    x = torch.zeros(3, 100, device=dev)
    tok = torch.zeros(3, dtype=torch.int32, device=dev)
    ok = dict(logits=x, tokens=tok, n_top=2)
    lstk.token_logprobs(**ok)
    bad = [dict(logits=x.half()), dict(logits=x.cpu()), dict(logits=x.t()), dict(logits=x[0]), dict(tokens=tok.long()), dict(tokens=tok[:2]),
           dict(tokens=tok.cpu()), dict(n_top=-1), dict(n_top=33), dict(n_top=2 ** 31), dict(logprobs=torch.zeros(2, device=dev)),
           dict(entropy=torch.zeros(3, dtype=torch.float64, device=dev)), dict(top_ids=torch.zeros(3, 3, dtype=torch.int32, device=dev)),
           dict(top_logprobs=torch.zeros(3, 2)), dict(logits=torch.zeros(1, 2 ** 20 - 15, device=dev), tokens=tok[:1]),
           dict(logits=x.expand(3, 100).as_strided((3, 100), (50, 1)))]
    for b in bad:
        with pytest.raises(lstk.LstkError) as e:
            lstk.token_logprobs(**{**ok, **b})
        assert e.value.code == lstk.E_INVALID, b
    big = torch.zeros(2, 50000, device=dev)
    with pytest.raises(lstk.LstkError):
        lstk.token_logprobs(big, tok[:2], n_top=2, work=torch.empty(16, dtype=torch.uint8, device=dev))
    r = lstk.token_logprobs(x[:0], tok[:0], n_top=4)
    assert [tuple(t.shape) for t in r] == [(0,), (0,), (0, 4), (0, 4)]
