"""Attention over the cache in 8 bits where scores are so large that their neighbours in fp32 lie far apart (2^18 to 2^30), beside V of any
scale: the largest cell alone counts, and its V comes out.

Tolerance: the other cells lie hundreds below, so the output is that V (d q, exact in fp32) off by a weight's two fp16 parts and the
quotient (2^-22 and 2 * 2^-24, below 2^-21 together), and by its rounding to fp16 (2^-11, or 2^-25 where it is subnormal)."""
import numpy as np
import pytest

import q8_cache as Q
from test_gpu_paged_attn_q8 import make

pytestmark = pytest.mark.gpu


def one_ahead(torch, dev, sign, scales, hd=64, n=200):
    """Scores of sign * (1/2 .. 1) of the largest in 64 steps, the last cell's above all others; blocks of V of the given scales."""
    c = make(torch, dev, np.random.default_rng(3), 2, 1, hd, [n])
    kd, kq, vd, vq = c["parts"]
    r = c["rows"][0]
    kd[0, r], kq[0, r] = np.float16(1.0), 0
    kq[0, r, 0, 0] = sign * np.linspace(64, 120, n)
    kq[0, r[-1], 0, 0] = 127 if sign > 0 else -60
    for m, s in enumerate(scales):
        vd[0, r, m] = np.float16(s)
    vq[0, r] = np.random.default_rng(4).integers(-127, 128, vq[0, r].shape)
    vq[0, r, 0] = np.where(vq[0, r, 0] % 2, 1, -1) if scales[0] > 100 else vq[0, r, 0]
    c["q"][:] = 0
    c["q"][:, :, 0] = 256.0
    c["qd"].copy_(torch.from_numpy(c["q"]))
    c["cache"].copy_(torch.from_numpy(Q.pack(*c["parts"])))
    return c, Q.values(vd, vq)[0, r[-1]]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("scales", [(0.02, 0.02), (2.0 ** -20, 0.5), (500.0, 2.0 ** -9), (40000.0, 0.01)])
def test_the_largest_cell_comes_out(lstk, dev, sign, scales):
    import torch
    c, want = one_ahead(torch, dev, sign, scales)
    tops = [2.0 ** 18, 2.0 ** 20 - 8, 2.0 ** 21, 2.0 ** 25, 2.0 ** 27] + [2.0e8 * (1 + 1.3e-7 * i) for i in range(12)] + [2.0 ** 29, 2.0 ** 30]
    for top in tops:
        got = lstk.paged_attention_q8(c["qd"], c["cache"], c["lens"], c["first"], c["blocks"], 200, scale=top / (256.0 * 127.0))
        got = got.float().cpu().numpy().astype(np.float64)[0]
        tol = np.abs(want) * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -25
        assert (np.abs(got - want) <= tol).all(), (top, float(np.abs(got - want).max()))


def test_a_block_of_nan_beside(lstk, dev):
    """A block of V that holds NaN leaves the other dims as they are, whatever the scores."""
    import torch
    c, want = one_ahead(torch, dev, 1, (0.02, 0.02))
    c["parts"][2][0, c["rows"][0][-1], 0] = np.nan
    c["cache"].copy_(torch.from_numpy(Q.pack(*c["parts"])))
    for top in [1.0e3, 2.0 ** 21] + [2.0e8 * (1 + 1.3e-7 * i) for i in range(12)]:
        got = lstk.paged_attention_q8(c["qd"], c["cache"], c["lens"], c["first"], c["blocks"], 200, scale=top / (256.0 * 127.0))
        got = got.float().cpu().numpy().astype(np.float64)[0]
        assert np.isnan(got[:, :32]).all()
        tol = np.abs(want[32:]) * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -25
        assert (np.abs(got[:, 32:] - want[32:]) <= tol).all(), (top, float(np.abs(got[:, 32:] - want[32:]).max()))
