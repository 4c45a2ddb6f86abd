"""Paged attention keeps its weights to 2^-22, like the attention of steps of one sequence: against the formula in 64 bits.

Tolerance, per output value, from the kernel's arithmetic (u16 = 2^-11, u32 = 2^-24, half steps of fp16 and fp32): a score is a
sum of head_dim products in fp32, off by at most E = (head_dim + 4) u32 sum_d |q_d k_d| scale, as is the largest one; a weight is
off by those, by its argument's rounding (2 u32 |s - max|, and 11 u32 for the 15 binary places that the maximum is lowered by), by
the exponential (2 u32) and as a sum of two fp16 parts by 2^-22 (of weights of up to 2^15; 2^-40 of the largest where the low part
is a subnormal fp16). The sums take two products a cell, so they are off by (2 n + 64) u32 each. The result's rounding is u16,
or half a subnormal step, 2^-25."""
import numpy as np
import pytest

from test_gpu_paged_attn import make

pytestmark = pytest.mark.gpu

U16, U32 = 2.0 ** -11, 2.0 ** -24


def formula(q, K, V, cells, scale):
    H, hd = q.shape
    out, tol = np.zeros((H, hd)), np.zeros((H, hd))
    for h in range(H):
        g = h // (H // K.shape[0])
        k, v, x = K[g, cells].astype(np.float64), V[g, cells].astype(np.float64), q[h].astype(np.float64)
        s = k @ x * scale
        e = (hd + 4) * U32 * (np.abs(k) @ np.abs(x)) * abs(scale)
        far = s.max() - s
        p = np.exp(-far)
        dp = p * (e + e[np.argmax(s)] + (13 + 2 * far) * U32 + 2.0 ** -22) + 2.0 ** -40
        t, a, n = p.sum(), np.abs(v), len(cells)
        out[h] = p @ v / t
        tol[h] = (dp @ a + np.abs(out[h]) * dp.sum()) / t + 2 * (2 * n + 64) * U32 * (p @ a) / t + U16 * np.abs(out[h]) + 2.0 ** -25
    return out, tol


def check(lstk, c, **kw):
    hd = c["q"].shape[2]
    got = lstk.paged_attention(c["qd"], c["kc"], c["vc"], c["lens"], c["first"], c["blocks"], c["max_len"], **kw)
    got = got.float().cpu().numpy().astype(np.float64)
    for b, cells in enumerate(c["rows"]):
        want, tol = formula(c["q"][b], c["K"], c["V"], cells, hd ** -0.5)
        err = np.abs(got[b] - want)
        assert (err <= tol).all(), (b, len(cells), int((err > tol).sum()), float((err / tol).max()))


def refill(torch, c):
    kv, size, hd = c["K"].shape
    c["kc"].copy_(torch.from_numpy(c["K"].reshape(kv, size, hd // 4, 4).transpose(0, 2, 1, 3).copy()))
    c["vc"].copy_(torch.from_numpy(c["V"].reshape(kv, size // 4, 4, hd).transpose(0, 1, 3, 2).copy()))
    c["qd"].copy_(torch.from_numpy(c["q"]))


@pytest.mark.parametrize("H,kv,hd", [(32, 4, 128), (4, 2, 64), (16, 2, 256), (40, 2, 128)])
def test_ordinary_weights(lstk, dev, H, kv, hd):
    """Weights of all sizes: most outputs are sums that nearly cancel, so a weight's own rounding shows."""
    import torch
    check(lstk, make(torch, dev, np.random.default_rng(H + hd), H, kv, hd, [40, 200, 97, 33, 1, 64, 500], spread=1.0))


def peaked(torch, dev, n, far, H=4, kv=1, hd=64):
    """One cell whose score is far natural units above all others', with V = 0; the others' V is 1000 and up."""
    c = make(torch, dev, np.random.default_rng(n), H, kv, hd, [n])
    r = c["rows"][0]
    c["K"][:, r] = 0
    c["K"][:, r[n // 3], 0] = 1.0
    c["q"][:] = 0
    c["q"][:, :, 0] = far * hd ** 0.5
    c["V"][:, r] = np.float16(1000.0) + np.arange(hd).astype(np.float16)
    c["V"][:, r[n // 3]] = 0
    refill(torch, c)
    return c


@pytest.mark.parametrize("bits", [8.0, 14.6, 20.5, 24.7, 26.3, 30.0])
@pytest.mark.parametrize("n", [100, 512, 3000])
def test_small_weights_count(lstk, dev, n, bits):
    """A cell 2^bits above all others (as a first cell often is): what the others add to the output is not lost."""
    import torch
    check(lstk, peaked(torch, dev, n, bits * np.log(2.0)))


def test_scores_too_large_to_be_lowered_exactly(lstk, dev):
    """Scores of 2^18 to 2^28, of both signs, whose neighbours lie hundreds apart: weights stay within fp16, and the largest
    cell's V comes out (its quotient is off by 2 u32, so it rounds to that V)."""
    import torch
    for top in (2.0 ** 18, 2.0 ** 20 - 8, 2.0 ** 21, 2.0 ** 25, 2.0 ** 28):
        for sign in (1.0, -1.0):
            c = make(torch, dev, np.random.default_rng(3), 2, 1, 64, [200])
            r = c["rows"][0]
            c["K"][:, r] = 0
            c["K"][0, r, 0] = sign * np.linspace(0.5, 1.0, 200).astype(np.float16)
            c["q"][:] = 0
            c["q"][:, :, 0] = 32768.0
            refill(torch, c)
            got = lstk.paged_attention(c["qd"], c["kc"], c["vc"], c["lens"], c["first"], c["blocks"], 200, scale=top / 32768.0)
            best = c["V"][0, r[-1 if sign > 0 else 0]]
            assert (got.cpu().numpy()[0] == best).all(), (top, sign)
