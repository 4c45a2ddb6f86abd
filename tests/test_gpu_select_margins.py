"""Groups whose two best choice values nearly cancel: a 32-bit sum is then off by the summands' roundings, not by its own, and the
pass in 64 bits has to decide. The rule in 64 bits with numpy is the oracle; both sides round the same sums, whose last bit is
2^-33 at a bias of 10^6, so scores that differ by a step of 2^-53 change none."""
import numpy as np
import pytest

from test_gpu_select import check, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,G,used,k", [(16, 8, 4, 4), (64, 8, 3, 6), (256, 8, 4, 8), (256, 128, 40, 8)])
@pytest.mark.parametrize("B", [1e2, 1e4, 1e5, 3e5, 1e6])
def test_biases_that_cancel(lstk, dev, E, G, used, k, B):
    """Two experts of each group have biases +B and -B, the others far less."""
    rng = np.random.default_rng(int(B) + E)
    per = E // G
    bias = np.full((G, per), -2 * B, np.float32)
    for g in range(G):
        a, b = rng.permutation(per)[:2]
        bias[g, a], bias[g, b] = B, -B
    x = logits(rng, 2000, E)
    check(lstk, dev, x, k, bias=bias.ravel(), score="sigmoid", n_group=G, n_group_used=used, group_top=2)
    check(lstk, dev, x, k, bias=bias.ravel(), score="softmax", n_group=G, n_group_used=used, group_top=2)


def test_close_groups(lstk, dev):
    """Groups of equal biases whose scores are a few 1e-7 apart, around what 32 bits can tell."""
    rng = np.random.default_rng(3)
    base = rng.standard_normal((500, 1, 8))
    x = (base + 10.0 ** rng.uniform(-8, -5, (500, 8, 1)) * rng.standard_normal((500, 8, 1))).reshape(500, 64).astype(np.float32)
    for top in (1, 2):
        for score in ("sigmoid", "softmax"):
            check(lstk, dev, x, 6, score=score, n_group=8, n_group_used=3, group_top=top)
