"""The numpy form of the 8-bit cache that the GPU tests compare with: its bounds, ties, and the layout's inverse (no GPU)."""
import numpy as np

import q8_cache as Q


def test_layout_has_an_inverse():
    rng = np.random.default_rng(1)
    for pages, kv, hd in ((1, 1, 64), (3, 2, 128), (2, 3, 256)):
        rec = rng.integers(0, 256, (pages, kv, 68 * hd), dtype=np.uint8)
        assert np.array_equal(Q.pack(*Q.unpack(rec)), rec)
        kd, kq, vd, vq = Q.unpack(rec)
        # byte by byte for a few places, from the format's text
        for p, g, cell, d in ((0, 0, 0, 0), (pages - 1, kv - 1, 31, hd - 1), (0, kv - 1, 13, 45), (pages - 1, 0, 22, 63)):
            m, x = d // 32, d % 32
            at = ((((m * 4 + x // 8) * 4 + cell // 8) * 4 + cell % 4) * 2 + cell // 4 % 2) * 8 + x % 8
            assert rec[p, g].view(np.int8)[at] == kq[g, 32 * p + cell, m, x]
            at = 34 * hd + (((m * 4 + cell // 8) * 16 + x % 16) * 2 + x // 16) * 8 + cell % 8
            assert rec[p, g].view(np.int8)[at] == vq[g, 32 * p + cell, m, x]
            assert rec[p, g].view(np.uint16)[16 * hd + 32 * m + cell] == kd.view(np.uint16)[g, 32 * p + cell, m]
            assert rec[p, g].view(np.uint16)[33 * hd + 32 * m + cell] == vd.view(np.uint16)[g, 32 * p + cell, m]


def test_rounding():
    rng = np.random.default_rng(2)
    for x in (rng.standard_normal((50, 64)), 1e-6 * rng.standard_normal((50, 64)), 1e5 * rng.standard_normal((50, 64)), np.zeros((1, 64)),
              np.full((1, 32), Q.MOST), np.full((1, 32), 2.0 ** -30)):
        x = x.astype(np.float32)
        d, q = Q.quantise(x)
        assert np.abs(q.astype(int)).max() <= 127
        off = np.abs(Q.values(d, q) - x).reshape(*d.shape, 32)
        assert (off <= d.astype(np.float64)[..., None] / 2).all()
        # the smallest such d: the fp16 number below it is less than a 127th of the largest
        below = np.nextafter(d, np.float16(0)).astype(np.float64)
        assert ((below * 127 < np.abs(x).reshape(*d.shape, 32).max(-1)) | (d == 0)).all()
    d, q = Q.quantise(np.array([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5] + [0.0] * 26], np.float32))
    assert d[0, 0] == 1 and q[0, 0, :6].tolist() == [127, 0, 2, 2, 0, -2]
    for bad in (np.nan, np.inf, -np.inf, 1.01 * Q.MOST):
        d, q = Q.quantise(np.array([[bad] + [1.0] * 63], np.float32))
        assert np.isnan(d[0, 0]) and float(d[0, 1]) * 127 >= 1 and not q[0, 0].any() and q[0, 1].all()
