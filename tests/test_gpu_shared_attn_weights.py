"""Attention over a shared prefix keeps its weights as lstk_attn_paged and lstk_attn_paged_q8 do, to 2^-22 each: against the formula in
64 bits over all of a sequence's cells.

Tolerance, per output value, from the kernels' arithmetic (u16 = 2^-11, u32 = 2^-24, half steps of fp16 and fp32). With `far` the
distance of a score below the largest: a score is a sum of head_dim products in fp32, off by at most E = (head_dim + 12) u32
sum_d |q_d k_d| scale (12: a quantised cell's scales, and the product with the scale where it is rounded), as is the largest one; the
scale times log2(e) is off by 2 u32, which shifts a weight by 2 u32 far; the exponential's argument lies within far log2(e) + 16, so its
rounding is u32 (far + 12); the exponential 2 u32; the sum of two fp16 parts 2^-22. Half a step of the subnormal numbers, 2^-25, is what a
small weight may be off by: the largest is 2^12 or more over the prefix and 2^15 over own fp16 cells (so 2^-37 of the largest, 2^-40 there);
over quantised cells it is a weight times a scale of V, 2^-38 times the scales' ratio (as test_gpu_paged_attn_q8.py has it), and the
product with the scale one more u32. The sums take two products a cell, so they are off by (2 n + 64) u32 each. The result's rounding is u16,
or half a subnormal step, 2^-25."""
import numpy as np
import pytest

import q8_cache as Q
from test_gpu_shared_attn import build, call

pytestmark = pytest.mark.gpu

U16, U32 = 2.0 ** -11, 2.0 ** -24


def formula(q, K, V, n_prefix, scale, spread=None):
    """(out, tolerance) of a sequence's heads over all cells, the prefix's first. spread: ratio of the own cells' scales of V."""
    H, hd = q.shape
    out, tol = np.zeros((H, hd)), np.zeros((H, hd))
    n = K.shape[1]
    for h in range(H):
        g = h // (H // K.shape[0])
        k, v, x = K[g], V[g], q[h].astype(np.float64)
        s = k @ x * scale
        e = (hd + 12) * U32 * (np.abs(k) @ np.abs(x)) * abs(scale)
        far = s.max() - s
        p = np.exp(-far)
        least = np.where(np.arange(n) < n_prefix, 2.0 ** -37, 2.0 ** -40 if spread is None else spread * 2.0 ** -38)
        dp = p * (e + e[np.argmax(s)] + (15 + 3 * far) * U32 + 2.0 ** -22) + least
        t, a = p.sum(), np.abs(v)
        out[h] = p @ v / t
        tol[h] = (dp @ a + np.abs(out[h]) * dp.sum()) / t + 2 * (2 * n + 64) * U32 * (p @ a) / t + U16 * np.abs(out[h]) + 2.0 ** -25
    return out, tol


def check(lstk, c, scale=None):
    hd, p = c["q"].shape[2], c["p"]
    got = call(lstk, c, scale=scale).float().cpu().numpy().astype(np.float64)
    spread = None
    if "cache" in c:
        d = Q.unpack(c["cache"].cpu().numpy())[2].astype(np.float64)
        held = d[np.isfinite(d) & (d > 0)]
        spread = held.max() / held.min() if held.size else 1.0
    for b, cells in enumerate(c["rows"]):
        K, V = (np.concatenate([a[:, p["cells"]].astype(np.float64), o[:, cells].astype(np.float64)], 1)
                for a, o in ((p["K"], c["K"]), (p["V"], c["V"])))
        want, tol = formula(c["q"][b], K, V, len(p["cells"]), hd ** -0.5 if scale is None else scale, spread)
        err = np.abs(got[b] - want)
        assert (err <= tol).all(), (b, len(cells), int((err > tol).sum()), float((err / tol).max()))


def refill(torch, c):
    """The fp16 caches and the queries of c once more, from its arrays."""
    for x in (c["p"], c):
        if "cache" in x:
            continue
        kv, size, hd = x["K"].shape
        x["kc"].copy_(torch.from_numpy(x["K"].astype(np.float16).reshape(kv, size, hd // 4, 4).transpose(0, 2, 1, 3).copy()))
        x["vc"].copy_(torch.from_numpy(x["V"].astype(np.float16).reshape(kv, size // 4, 4, hd).transpose(0, 1, 3, 2).copy()))
    c["qd"].copy_(torch.from_numpy(c["q"]))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("H,kv,hd", [(32, 4, 128), (4, 2, 64), (16, 2, 256), (40, 2, 128)])
@pytest.mark.parametrize("n,prefix", [(1, 33), (2, 700), (20, 200), (36, 1055)])
def test_ordinary_weights(lstk, dev, H, kv, hd, n, prefix, bits):
    """Weights of all sizes, over the prefix and over own cells: most outputs are sums that nearly cancel, so a weight's own rounding shows."""
    import torch
    rng = np.random.default_rng(H + hd + prefix)
    check(lstk, build(torch, dev, rng, H, kv, hd, prefix, rng.integers(0, 70, n).tolist(), spread=1.0, bits=bits))


@pytest.mark.parametrize("where", ["prefix", "own", "own in 8 bits"])
@pytest.mark.parametrize("n", [2, 20])
def test_values_that_cancel(lstk, dev, n, where):
    """32 cells of V = 1000 at the largest weight and 32 of V = -1000 at one a little below it, the same for all of them, so that its rounding
    does not average out: a weight in one fp16 part puts the output off by up to 1000 * 2^-13, over twice the tolerance."""
    import torch
    c = build(torch, dev, np.random.default_rng(n), 8, 1, 64, 64, [64] * n, bits=8 if "8" in where else 16)
    p, cells, own = c["p"], c["p"]["cells"], np.concatenate(c["rows"])
    near, far = ((p, cells), (c, own)) if where == "prefix" else ((c, own), (p, cells))
    sides = np.arange(len(near[1])) % 2 == 1
    if "cache" in c:
        kd, kq, vd, vq = Q.unpack(c["cache"].cpu().numpy())
        kd[0, own], vd[0, own] = 2.0 ** -6, 8.0
        kq[0, own], vq[0, own] = 0, np.where(sides, 125, -125)[:, None, None]
        kq[0, own, 0, 0] = np.where(sides, 0, -64)
        with np.errstate(invalid="ignore"):
            c["K"], c["V"] = Q.values(kd, kq), Q.values(vd, vq)
        c["cache"].copy_(torch.from_numpy(Q.pack(kd, kq, vd, vq)))
    else:
        near[0]["K"][0, near[1]] = 0
        near[0]["K"][0, near[1], 0] = np.where(sides, 0.0, -1.0)
        near[0]["V"][0, near[1]] = np.where(sides, 1000.0, -1000.0)[:, None]
    far[0]["K"][0, far[1]] = 0
    far[0]["K"][0, far[1], 0] = -60000.0
    c["q"][:] = 0
    c["q"][:, :, 0] = np.linspace(0.01, 0.05, 8 * n).reshape(n, 8).astype(np.float16)
    refill(torch, c)
    check(lstk, c, scale=1.0)


@pytest.mark.parametrize("n", [2, 20])
@pytest.mark.parametrize("bits", [8.0, 14.6, 20.5, 24.7, 26.3, 30.0])
def test_small_weights_count(lstk, dev, n, bits):
    """A cell of the prefix 2^bits above all others (as a first cell often is), with V = 0: what the others add is not lost."""
    import torch
    for prefix in (100, 3000):
        c = build(torch, dev, np.random.default_rng(n), 4, 1, 64, prefix, [50, 0] * (n // 2))
        p, cells, own = c["p"], c["p"]["cells"], np.concatenate(c["rows"])
        for x, at in ((p, cells), (c, own)):
            x["K"][:, at] = 0
            x["V"][:, at] = np.float16(1000.0) + np.arange(64).astype(np.float16)
        p["K"][:, cells[prefix // 3], 0] = 1.0
        p["V"][:, cells[prefix // 3]] = 0
        c["q"][:] = 0
        c["q"][:, :, 0] = bits * np.log(2.0) * 8.0
        refill(torch, c)
        check(lstk, c)
