"""Log probabilities and entropies of rows that one token nearly has to itself: small numbers, right relative to themselves.

With z = x - max over the row's other values, S = sum e^z over them and k values at the maximum: ln l = log1p(k - 1 + S), for k = 1 about S.
Tolerance, from the kernel's arithmetic (u = 2^-24): a term of S is off by (2 + 2 |z|) u relative (the difference's rounding, its product
with log2 e and that constant's own rounding; the exponential), a thread's sum of up to 64 of them and its wavefront's by (64 + 8) u, a
slice's share of it as fp32 by u: with D = sum e^z |z| / S that is (75 + 2 D) u of S, and log1p passes a relative error on. A result
is rounded once more. The entropy is ln l + sum e^z |z| / l; a term of that sum is off by (3 + 3 |z|) u (z's rounding and the product
besides), so the sum by (76 u) of itself and 3 u sum e^z z^2. Terms below 2^-126 are 0."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def expect(x):
    x = x.astype(np.float64)
    z = x - x.max(1, keepdims=True)
    rest = z < 0
    w = np.where(rest, np.exp(z), 0.0)
    zf = np.where(w > 0, z, 0.0)  # (-inf has no part)
    S, k = w.sum(1), (~rest).sum(1)
    first, second = (w * np.abs(zf)).sum(1), (w * zf * zf).sum(1)
    lse = np.log1p(k - 1 + S)
    lost = x.shape[1] * 2.0 ** -126 * 100
    tol_l = 76 * U * S + 2 * U * first + U * lse + lost
    l = k + S
    tol_e = tol_l + (77 * U * first + 3 * U * second) / l + first * (76 * U * S + 2 * U * first) / l ** 2 + 2 * U * (lse + first / l) + lost
    return lse, lse + first / l, tol_l, tol_e


def check(lstk, dev, x, n_top=3):
    import torch
    at = x.argmax(1).astype(np.int32)
    other = (at + 1) % x.shape[1]
    lse, entropy, tol_l, tol_e = expect(x)
    xd = torch.from_numpy(x).to(dev)
    for tokens in (at, other):
        of, ent, ids, top = (t.cpu().numpy().astype(np.float64) for t in lstk.token_logprobs(xd, torch.from_numpy(tokens).to(dev), n_top=n_top))
        z = x[np.arange(len(x)), tokens].astype(np.float64) - x.max(1).astype(np.float64)
        want = z - lse
        assert (np.abs(of - want) <= tol_l + U * np.abs(want)).all(), (of, want)
        assert (np.abs(ent - entropy) <= tol_e).all(), (ent, entropy)
        if n_top:
            assert np.array_equal(ids[:, 0], at) and (np.abs(top[:, 0] + lse) <= tol_l).all()


@pytest.mark.parametrize("V", [2, 50, 1024, 5000, 50259, 151936])
@pytest.mark.parametrize("n_top", [0, 3])
def test_one_token_ahead(lstk, dev, V, n_top):
    rng = np.random.default_rng(V)
    ahead = [1.0, 8.0, 14.0, 17.0, 20.0, 30.0, 45.0, 70.0]
    x = (2.0 * rng.standard_normal((len(ahead), V))).astype(np.float32)
    for r, d in enumerate(ahead):
        x[r, (r * 7919 + 3) % V] = x[r].max() + np.float32(d)
    check(lstk, dev, x, n_top)
    x[:, V // 2] = -np.inf if V > 2 else x[:, V // 2]
    x[np.arange(len(ahead)), np.arange(len(ahead)) * 7919 % V] += 0.0
    check(lstk, dev, x, n_top)


@pytest.mark.parametrize("rows", [1, 64, 500])
def test_rows_of_slices_and_of_few(lstk, dev, rows):
    """Rows in many slices, in few and in one, a work-group's share with the largest value or without."""
    rng = np.random.default_rng(rows)
    x = (1.5 * rng.standard_normal((rows, 20003))).astype(np.float32)
    x[np.arange(rows), rng.integers(0, 20003, rows)] = x.max(1) + (5.0 + 40.0 * rng.random(rows)).astype(np.float32)
    check(lstk, dev, x)


def test_two_and_more_at_the_maximum(lstk, dev):
    """k values alike far above the others: ln k and a little, in one slice and over several."""
    rng = np.random.default_rng(1)
    for V in (300, 60000):
        x = (2.0 * rng.standard_normal((4, V))).astype(np.float32)
        for r, k in enumerate((2, 3, 40, 299)):
            x[r, rng.choice(V, k, replace=False)] = 60.0
        check(lstk, dev, x)


def test_nothing_but_one(lstk, dev):
    """All other values at -inf: log probability and entropy are 0."""
    import torch
    x = torch.full((2, 40000), -np.inf, device=dev)
    x[0, 17], x[1, 39999] = 3.0, -5.0
    of, ent, ids, top = lstk.token_logprobs(x, torch.tensor([17, 39999], dtype=torch.int32, device=dev), n_top=2)
    assert not of.any() and not ent.any() and ids.tolist() == [[17, -1], [39999, -1]] and not top[:, 0].any()
