"""The 8-bit cache in numpy, from its documented format (include/lstk_qwen3.h), in 64 bits."""
import numpy as np

MOST = 65504.0 * 127.0  # the largest magnitude that a block holds


def quantise(x):
    """(d fp16 [..., hd / 32], q int8 [..., hd / 32, 32]) of rows [..., hd] of fp16 or f32."""
    x = np.asarray(x).astype(np.float64)
    x = x.reshape(*x.shape[:-1], -1, 32)
    most = np.abs(x).max(-1)
    bad = ~(most <= MOST)
    a = np.where(bad, 0.0, most)
    d = (a / 127).astype(np.float16)
    with np.errstate(over="ignore"):  # (of the largest, which is not taken)
        d = np.where(d.astype(np.float64) * 127 < a, np.nextafter(d, np.float16(np.inf)), d)
    step = np.where(d == 0, 1.0, d.astype(np.float64))[..., None]
    q = np.rint(np.where(bad[..., None], 0.0, x) / step).astype(np.int8)
    return np.where(bad, np.float16(np.nan), d).astype(np.float16), q


def values(d, q):
    """d q in 64 bits, [..., hd]."""
    with np.errstate(invalid="ignore"):
        v = d.astype(np.float64)[..., None] * q.astype(np.float64)
    return v.reshape(*v.shape[:-2], -1)


def pack(kd, kq, vd, vq):
    """The bytes [pages][kv][68 hd] of K and V as [kv][cells][hd / 32] scales and [kv][cells][hd / 32][32] numbers."""
    kv, cells, m, _ = kq.shape
    pages, hd = cells // 32, 32 * m
    byte = lambda a: np.ascontiguousarray(a).reshape(pages, kv, -1).view(np.uint8).reshape(pages, kv, -1)
    # [kv][page][b][t][c][m][a][j] -> [page][kv][m][a][b][c][t][j]
    k = kq.reshape(kv, pages, 4, 2, 4, m, 4, 8).transpose(1, 0, 5, 6, 2, 4, 3, 7)
    # [kv][page][a][c][m][t][r] -> [page][kv][m][a][r][t][c]
    v = vq.reshape(kv, pages, 4, 8, m, 2, 16).transpose(1, 0, 4, 2, 6, 5, 3)
    scale = lambda d: d.reshape(kv, pages, 32, m).transpose(1, 0, 3, 2)
    return np.concatenate([byte(k), byte(scale(kd)), byte(v), byte(scale(vd))], 2)


def unpack(rec):
    """The inverse of pack: (kd, kq, vd, vq)."""
    pages, kv, n = rec.shape
    hd = n // 68
    m, cells = hd // 32, 32 * pages
    part = lambda a, b, t: np.ascontiguousarray(rec[:, :, a * hd:b * hd]).view(t)
    kq = part(0, 32, np.int8).reshape(pages, kv, m, 4, 4, 4, 2, 8).transpose(1, 0, 4, 6, 5, 2, 3, 7).reshape(kv, cells, m, 32)
    vq = part(34, 66, np.int8).reshape(pages, kv, m, 4, 16, 2, 8).transpose(1, 0, 3, 6, 2, 5, 4).reshape(kv, cells, m, 32)
    scale = lambda a, b: part(a, b, np.float16).reshape(pages, kv, m, 32).transpose(1, 0, 3, 2).reshape(kv, cells, m)
    return scale(32, 34), kq, scale(66, 68), vq
