"""Sampling of the next token (lstk_sample) against a sort in 64 bits.

Tokens have to be equal: the running sums that decide are whole numbers on the device (each weight rounded to 2^-44 of the
largest) and 64-bit sums here, so they differ by less than n 2^-45 of the largest weight, and the seeds' draws lie further
from every border than that (asserted). The probability is a quotient of the two, rounded to fp32: off by 2^-24 relative,
and n 2^-45 over the sum of what stays (at least 1)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FMAX = np.finfo(np.float32).max


def pick(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """(token, probability, distance of the draw and of the top-p cut from the next border)."""
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, FMAX)).astype(np.float64)
    if not np.isfinite(x.max()):
        return -1, 0.0, 1.0
    if not T > 0:
        return int(np.argmax(x)), 1.0, 1.0
    order = np.argsort(-x, kind="stable")
    order = order[np.isfinite(x[order])]
    with np.errstate(over="ignore", under="ignore"):
        w = np.exp((x[order] - x.max()) / np.float64(np.float32(T)))
    if k > 0:
        order, w = order[:k], w[:k]
    n = max(1, int((w >= min(np.float64(np.float32(m)), 1.0)).sum())) if m > 0 else len(w)
    order, w = order[:n], w[:n]
    gap = 1.0
    p = np.float64(np.float32(p))
    if p < 1:
        cum = np.cumsum(w)
        t = max(p, 0.0) * cum[-1]
        n = int(np.searchsorted(cum, t, side="left")) + 1
        gap = np.abs(cum - t)[w > 2.0 ** -40].min()
        order, w = order[:n], w[:n]
    cum = np.cumsum(w)
    u = 0.0 if not u > 0 else float(u)
    i = min(int(np.searchsorted(cum, u * cum[-1], side="right")), int((w > 2.0 ** -45).sum()) - 1)
    if 0 < u < 1:
        gap = min(gap, np.abs(cum - u * cum[-1])[w > 2.0 ** -40].min())
    return int(order[i]), w[i] / cum[-1], gap


def check(lstk, dev, x, u, T=None, k=None, p=None, m=None, borders=False, xd=None):
    import torch
    d = lambda a, t: None if a is None else torch.tensor(np.asarray(a, t), device=dev)
    xd = d(x, np.float32) if xd is None else xd
    n, V = x.shape
    full = lambda a, v: np.full(n, v) if a is None else np.asarray(a)
    tok, prob = lstk.sample(xd, d(u, np.float32), temperature=d(T, np.float32), top_k=d(k, np.int32), top_p=d(p, np.float32),
                            min_p=d(m, np.float32))
    tok, prob = tok.cpu().numpy(), prob.cpu().numpy()
    T, k, p, m = full(T, 1.0), full(k, 0), full(p, 1.0), full(m, 0.0)
    for r in range(n):
        pr, mr = (1.0 if np.isnan(p[r]) else p[r]), (0.0 if np.isnan(m[r]) else m[r])
        want, wp, gap = pick(x[r], u[r], T[r], k[r], pr, mr)
        if not borders:
            assert gap > V * 2.0 ** -44, (r, gap)  # the seed's draw is no border case
        assert tok[r] == want, (r, tok[r], want, T[r], k[r], p[r], m[r], u[r])
        assert abs(prob[r] - wp) <= wp * 2.0 ** -24 + V * 2.0 ** -44, (r, prob[r], wp)
    return tok, prob


def logits(rng, n, V, sd=2.5):
    x = sd * rng.standard_normal((n, V))
    for r in range(n):
        at = rng.permutation(V)[:min(V, 200)]
        x[r, at] += 12 - (0.5 + r % 3) * np.log(np.arange(1, len(at) + 1))
    return x.astype(np.float32)


SETTINGS = [(0.7, 20, 0.8, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.95, 0.0), (0.6, 0, 1.0, 0.1), (1.3, 1000, 0.99, 0.01), (1.0, 0, 1.0, 0.0),
            (0.8, 50, 1.0, 0.0), (2.5, 0, 0.5, 0.0), (0.05, 0, 0.9, 0.0), (5.0, 100000, 0.999, 1e-6), (1.0, 1, 1.0, 0.0),
            (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (-1.0, 5, 0.5, 0.5)]


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 4095, 4096, 4097, 50257, 151936, 262144])
def test_settings_and_sizes(lstk, dev, V):
    rng = np.random.default_rng(V)
    n = 2 * len(SETTINGS)
    s = SETTINGS * 2
    check(lstk, dev, logits(rng, n, V), rng.random(n).astype(np.float32), *[[r[i] for r in s] for i in range(4)])


@pytest.mark.parametrize("n", [1, 3, 130, 700])
def test_rows(lstk, dev, n):
    rng = np.random.default_rng(n)
    s = [SETTINGS[i % len(SETTINGS)] for i in range(n)]
    check(lstk, dev, logits(rng, n, 5001), rng.random(n).astype(np.float32), *[[r[i] for r in s] for i in range(4)])


def test_no_settings(lstk, dev):
    rng = np.random.default_rng(1)
    check(lstk, dev, logits(rng, 9, 32000), rng.random(9).astype(np.float32))


def test_equal_values(lstk, dev):
    """Rows of equal values, and of a few values many times over: the lowest index comes first, borders are exact."""
    for V in (5, 1000, 151936):
        x = np.zeros((6, V), np.float32)
        x[3:] = (np.arange(V) % 3).astype(np.float32)
        u = np.array([0.0, 0.5, 1 - 2.0 ** -24] * 2, np.float32)
        check(lstk, dev, x, u, borders=True)
        check(lstk, dev, x, u, p=[0.5] * 6, borders=True)
        check(lstk, dev, x, u, k=[V // 2 + 1] * 6, borders=True)
        check(lstk, dev, x, u, k=[V // 2 + 1] * 6, p=[0.25] * 6, m=[0.5] * 6, borders=True)
    x = np.full((1, 9), -0.0, np.float32)
    x[0, 4:] = 0.0  # 0 and -0 are equal
    check(lstk, dev, x, [0.0], k=[3], borders=True)


@pytest.mark.parametrize("n,V", [(3, 1024), (3, 1025), (2, 16384), (2, 16385), (97, 40000), (96, 49149), (96, 49150)])
def test_many_equal_values_in_one_row(lstk, dev, n, V):
    """More values where a cut falls than are sorted, with one work-group to a row and with several, at the sizes where that and
    the row's place in registers change."""
    rng = np.random.default_rng(V)
    x = np.zeros((n, V), np.float32)
    x[::2] = (rng.integers(0, 3, V) / 7).astype(np.float32)
    x[0] = 2.2 * rng.standard_normal(V).astype(np.float32)
    u = rng.random(n).astype(np.float32)
    check(lstk, dev, x, u, borders=True)
    check(lstk, dev, x, u, k=[V // 2 + 3] * n, p=[0.625] * n, borders=True)
    check(lstk, dev, x, u, p=[0.5] * n, m=[0.25] * n, borders=True)


def test_special_values(lstk, dev):
    inf, nan = np.inf, np.nan
    rows = [[-inf] * 6, [nan] * 6, [-inf, nan, -inf, 3.0, nan, -inf], [1, nan, 2, -inf, 0, 1], [inf, 1, 2, inf, 3, -inf], [FMAX, inf, -FMAX, 0, 1, 2],
            [-FMAX, -FMAX, -inf, nan, -FMAX, -inf], [1e-38, 0, -1e-38, 2e-38, 0, 0]]
    x = np.array(rows, np.float32)
    n = len(rows)
    for u in (0.0, 0.3, 0.99):
        check(lstk, dev, x, [u] * n, borders=True)
        check(lstk, dev, x, [u] * n, k=[2] * n, p=[0.9] * n, borders=True)
        check(lstk, dev, x, [u] * n, T=[0.0] * n, borders=True)


def test_special_settings(lstk, dev):
    rng = np.random.default_rng(4)
    x = logits(rng, 1, 3000)
    inf, nan = np.inf, np.nan
    for T in (nan, inf, 1e-30, 1e-45, 1e30, -inf):
        check(lstk, dev, x, [0.4], T=[T], borders=True)
    for p in (nan, -1.0, 2.0, 1e-30, 1 - 2.0 ** -24, inf):
        check(lstk, dev, x, [0.4], p=[p], borders=True)
    for m in (nan, -1.0, 2.0, 1e-30, inf):
        check(lstk, dev, x, [0.4], m=[m], borders=True)
    for k in (-5, 2 ** 31 - 1, 3000, 2999):
        check(lstk, dev, x, [0.4], k=[k], borders=True)
    for u in (nan, -1.0, 0.0, 1.0, 5.0):
        import torch
        t, _ = lstk.sample(torch.tensor(x, device=dev), torch.tensor([u], device=dev), top_k=torch.tensor([7], dtype=torch.int32, device=dev))
        order = np.argsort(-x[0], kind="stable")
        assert int(t) == (order[6] if u >= 1 else order[0]), u


def test_every_quantile(lstk, dev):
    """One row drawn with many numbers: the tokens come in order, each as often as its probability says."""
    rng = np.random.default_rng(6)
    n = 512
    x = np.repeat(logits(rng, 1, 20000), n, 0)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    check(lstk, dev, x, u, T=[0.8] * n, p=[0.97] * n)


def test_strided_and_unaligned_rows(lstk, dev):
    import torch
    rng = np.random.default_rng(7)
    x = logits(rng, 5, 10007)
    for off, ld in ((0, 10240), (1, 10008), (3, 11111)):
        big = torch.full((5, ld + off), 50.0, device=dev)
        view = big[:, off:off + 10007]
        view.copy_(torch.from_numpy(x))
        check(lstk, dev, x, rng.random(5).astype(np.float32), p=[0.9] * 5, xd=view)


def test_repeats_and_rows_behind_stay(lstk, dev):
    import torch
    rng = np.random.default_rng(8)
    x, u = torch.from_numpy(logits(rng, 6, 60000)).to(dev), torch.rand(6, device=dev)
    need = lstk.sample_work_bytes(4, 60000)
    work = torch.full((need + 64,), 9, dtype=torch.uint8, device=dev)
    tok, prob = torch.full((6,), -9, dtype=torch.int32, device=dev), torch.full((6,), -9.0, device=dev)
    first = None
    for _ in range(5):
        lstk.sample(x[:4], u[:4], tokens=tok[:4], probs=prob[:4], work=work[:need])
        got = (tok.tolist(), prob.tolist())
        first = first or got
        assert got == first
    assert first[0][4:] == [-9, -9] and first[1][4:] == [-9.0, -9.0] and (work[need:] == 9).all()


def test_capture_and_stream(lstk, dev):
    import torch
    rng = np.random.default_rng(9)
    x, u = torch.from_numpy(logits(rng, 8, 151936)).to(dev), torch.rand(8, device=dev)
    T = torch.tensor([0.0, 0.7, 1.0, 1.2] * 2, device=dev)
    p = torch.full((8,), 0.9, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = lstk.sample(x, u, temperature=T, top_p=p, stream=side)
    side.synchronize()
    b = lstk.sample(x, u, temperature=T, top_p=p)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    work = torch.empty(lstk.sample_work_bytes(8, 151936), dtype=torch.uint8, device=dev)
    tok, prob = torch.zeros(8, dtype=torch.int32, device=dev), torch.zeros(8, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lstk.sample(x, u, temperature=T, top_p=p, tokens=tok, probs=prob, work=work)
    for step in range(5):
        x.mul_(0.9)
        u.copy_(torch.from_numpy(rng.random(8).astype(np.float32)))
        T.copy_(T.roll(1))
        g.replay()
        ref = lstk.sample(x, u, temperature=T, top_p=p)
        assert torch.equal(tok, ref[0]) and torch.equal(prob, ref[1]), step


def test_refusals_of_tensors(lstk, dev):
    import torch
    x, u = torch.zeros(3, 50, device=dev), torch.zeros(3, device=dev)
    lstk.sample(x, u)
    f, i = torch.zeros(3, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    for kw in (dict(logits=x.half()), dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=x.t()), dict(u=u.double()), dict(u=u[:2]),
               dict(u=u.cpu()), dict(top_k=f), dict(temperature=i), dict(top_p=f[:2]), dict(min_p=f.cpu()), dict(tokens=f), dict(probs=i),
               dict(work=torch.empty(10, dtype=torch.uint8, device=dev)), dict(logits=x.expand(3, 50)[:1].expand(3, 50)),
               dict(logits=torch.zeros(3, 0, device=dev))):
        with pytest.raises(lstk.LstkError) as e:
            lstk.sample(**{**dict(logits=x, u=u), **kw})
        assert e.value.code == lstk.E_INVALID, kw
    t, p = lstk.sample(x[:0], u[:0])
    assert t.numel() == 0 and p.numel() == 0


def test_new_tensors_are_of_the_given_stream(lstk, dev):
    """What a call allocates for another stream is not memory that the current stream has just freed (its kernels may still be
    at work there), whether the stream comes as an object or as a handle."""
    import torch
    x, u = torch.zeros(4, 20000, device=dev), torch.zeros(4, device=dev)
    sizes = (lstk.sample_work_bytes(4, 20000), 16, 16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream):
        freed = [torch.empty(n, dtype=torch.uint8, device=dev) for n in sizes for _ in range(2)]
        at = {t.data_ptr() for t in freed}
        del freed
        work = lstk._work(None, sizes[0], 0, stream)[0]
        tokens, probs = lstk.sample(x, u, work=work, stream=stream)
        side.synchronize()
        assert not at & {t.data_ptr() for t in (work, tokens, probs)}
        assert (tokens == 0).all()
    work = lstk._work(None, sizes[0], 0, 0)[0]  # the null stream's handle
    assert (lstk.sample(x, u, work=work, stream=0)[0].cpu() == 0).all()
