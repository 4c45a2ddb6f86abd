"""Routing orders choice values by all their 64 bits: ones a few steps of 2^-53 apart are not equal.

The rule in 64 bits with numpy is the oracle. The kernel's sigmoid is 1 / (1 + t) with t = e^-x good to 1e-15 of itself and the
quotient rounded to nearest, so where t is small it has numpy's bits unless t lies within 1e-15 t of the middle between two
neighbouring sums; softmax scores far below 1 are off by a few 1e-16 of themselves, and the sum with a bias rounds that away."""
import numpy as np
import pytest

from test_gpu_select import check, rule_of

pytestmark = pytest.mark.gpu

# sigmoids 4 steps of 2^-53 apart and more
SATURATED = np.array([20, 22.5, 25, 25.001, 26, 27, 28, 29, 30, 30.5, 31, 31.5, 32, 32.5, 33, 33.5, 34, 34.5], np.float32)


def test_two_saturated_sigmoids(lstk, dev):
    """The larger one has the higher id."""
    for a, b in ((33, 34), (33, 36), (25, 25.001), (30, 40)):
        x = np.array([[a, b], [b, a]], np.float32)
        ids, _ = check(lstk, dev, x, 1, score="sigmoid")
        assert ids.cpu().numpy().ravel().tolist() == [1, 0]
        check(lstk, dev, np.concatenate([x, np.full((2, 62), -3, np.float32)], 1), 2, score="sigmoid")


@pytest.mark.parametrize("E", [24, 64, 128, 200, 256])
@pytest.mark.parametrize("bias", [False, True])
def test_saturated_sigmoids(lstk, dev, E, bias):
    """All of SATURATED at random experts: more than are candidates, so that the pass in 64 bits chooses; with a bias that is
    alike for all (1 / 8: the sum keeps all but three bits, the values stay 2^-53 apart or more)."""
    assert (np.diff(1 / (1 + np.exp(-SATURATED.astype(np.float64)))) >= 4 * 2.0 ** -53).all()
    rng = np.random.default_rng(E)
    x = np.full((40, E), -2.0, np.float32)
    for t in range(40):
        x[t, rng.permutation(E)[:len(SATURATED)]] = SATURATED
    b = np.full(E, 0.125, np.float32) if bias else None
    for k in (1, 5, 8, 18):
        check(lstk, dev, x, k, bias=b, score="sigmoid")
        check(lstk, dev, x, min(k, E // 2), bias=b, score="sigmoid", n_group=4, n_group_used=2, group_top=1)


def test_few_saturated_sigmoids(lstk, dev):
    """Few enough that all are candidates of the 32-bit pass, which then orders them."""
    rng = np.random.default_rng(7)
    x = np.full((64, 128), -2.0, np.float32)
    for t in range(64):
        x[t, rng.permutation(128)[:8]] = rng.permutation(SATURATED)[:8]
    for k in (5, 6, 8):
        check(lstk, dev, x, k, score="sigmoid")


@pytest.mark.parametrize("E,k", [(256, 8), (64, 6)])
def test_wide_sigmoid_logits(lstk, dev, E, k):
    """Logits of standard deviation 12: some of every fourth row's best lie in the saturated range."""
    x = (12 * np.random.default_rng(E).standard_normal((400, E))).astype(np.float32)
    check(lstk, dev, x, k, score="sigmoid")
    check(lstk, dev, x, k, score="sigmoid", n_group=8, n_group_used=4, group_top=2)


@pytest.mark.parametrize("E", [16, 64, 256])
def test_peaked_softmax_with_a_bias(lstk, dev, E):
    """One expert has nearly all of the softmax; the others' scores of 1e-15 to 1e-13 on a bias of 1 / 2 are all that tells them
    apart (the sum's last bit is 2^-53)."""
    rng = np.random.default_rng(E)
    x = np.stack([rng.permutation(np.linspace(-33.5, -30, E)) for _ in range(50)]).astype(np.float32)
    x[np.arange(50), rng.integers(0, E, 50)] = 0
    want, _ = rule_of(x, 6, bias=np.full(E, 0.5, np.float32))
    assert (np.sort(want, 1) != want).any(1).mean() > 0.8  # the order is not that of the ids
    check(lstk, dev, x, 6, bias=np.full(E, 0.5, np.float32))
    check(lstk, dev, x, 4, bias=np.full(E, 0.5, np.float32), renorm=False, n_group=4, n_group_used=2, group_top=2)
