"""Rows quantised as they are written to a cache in 8 bits, and read back, bit for bit against the format in 64 bits."""
import numpy as np
import pytest

import q8_cache as Q

pytestmark = pytest.mark.gpu

HEADS = [(4, 128), (2, 64), (2, 256), (1, 64), (3, 128)]


def cells_of(rng, n, pages, how):
    """n different cells: in a row from an odd place on over pages in any order, backwards, or anywhere."""
    if how == "any":
        return rng.permutation(32 * pages)[:n]
    order = rng.permutation(pages)
    i = np.arange(n) + {"row": 0, "row13": 13, "row7": 7, "back": 5}[how]
    c = order[i // 32] * 32 + i % 32
    return c[::-1].copy() if how == "back" else c


def rows_of(rng, n, kv, hd, dtype, spread=1.0):
    x = spread * rng.standard_normal((n, 2, kv, hd)) * np.exp(rng.standard_normal((1, 2, kv, hd)))
    return x.astype(dtype)


def expect(rec, rows, cells):
    """The cache's bytes after these rows went to these cells."""
    kd, kq, vd, vq = (a.copy() for a in Q.unpack(rec))
    inside = (cells >= 0) & (cells < kq.shape[1])
    for x, d, q in ((rows[:, 0], kd, kq), (rows[:, 1], vd, vq)):
        d2, q2 = Q.quantise(x[inside])
        d[:, cells[inside]], q[:, cells[inside]] = d2.transpose(1, 0, 2), q2.transpose(1, 0, 2, 3)
    return Q.pack(kd, kq, vd, vq)


def run(lstk, dev, rng, rows, cells, pages, **kw):
    import torch
    n, _, kv, hd = rows.shape
    rec = rng.integers(0, 256, (pages, kv, 68 * hd), dtype=np.uint8)
    cache, r = torch.from_numpy(rec).to(dev), torch.from_numpy(rows).to(dev)
    at = torch.tensor(cells, dtype=torch.int32, device=dev)
    lstk.store_q8(cache, r[:, 0], r[:, 1], at, **kw)
    got = cache.cpu().numpy()
    want = expect(rec, rows, cells)
    # a block that does not fit is any NaN
    g, w = Q.unpack(got), Q.unpack(want)
    for i in (0, 2):
        nan = np.isnan(w[i])
        old = np.isnan(g[i])
        assert np.array_equal(nan, old)
        assert np.array_equal(g[i].view(np.uint16)[~nan], w[i].view(np.uint16)[~nan]), "scales"
    assert np.array_equal(g[1], w[1]), "K"
    assert np.array_equal(g[3], w[3]), "V"
    return cache, at, got


def check_back(lstk, dev, cache, at, got, dtypes=(np.float16, np.float32)):
    import torch
    kd, kq, vd, vq = Q.unpack(got)
    cells = at.cpu().numpy()
    inside = (cells >= 0) & (cells < kq.shape[1])
    for dtype in dtypes:
        out = lstk.load_q8(cache, at, dtype=torch.float16 if dtype is np.float16 else torch.float32)
        for x, d, q in zip(out, (kd, vd), (kq, vq)):
            with np.errstate(over="ignore"):
                want = np.zeros(x.shape, dtype)
                want[inside] = Q.values(d, q)[:, cells[inside]].transpose(1, 0, 2).astype(dtype)
            x = x.cpu().numpy()
            assert x.dtype == dtype and np.array_equal(np.isnan(x), np.isnan(want))
            assert np.array_equal(x[~np.isnan(x)], want[~np.isnan(want)])


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("kv,hd", HEADS)
@pytest.mark.parametrize("n,how", [(1, "any"), (1, "row7"), (8, "row"), (31, "row"), (32, "any"), (33, "row13"), (77, "back"), (100, "row7"),
                                   (203, "row13"), (300, "any")])
def test_store_and_load(lstk, dev, dtype, kv, hd, n, how):
    rng = np.random.default_rng(n * hd + kv)
    pages = -(-(n + 16) // 32) + 2
    cache, at, got = run(lstk, dev, rng, rows_of(rng, n, kv, hd, dtype), cells_of(rng, n, pages, how), pages)
    check_back(lstk, dev, cache, at, got)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_halves_and_ends(lstk, dev, dtype):
    """Values exactly between two whole numbers, blocks of zeros, of subnormal scales, of one large dim, and of the largest numbers."""
    rng = np.random.default_rng(5)
    n, kv, hd = 64, 2, 128
    rows = rows_of(rng, n, kv, hd, np.float64)
    d = rng.integers(1024, 2048, (n, 2, kv, hd // 32, 1)).astype(np.float64) * 2.0 ** -14  # an 11-bit scale
    t = d * (rng.integers(-126, 127, (n, 2, kv, hd // 32, 32)) + 0.5)
    t[..., 0] = 127 * d[..., 0]  # the largest of a block gives just this d (18 bits)
    half = t.reshape(n, 2, kv, hd)
    rows[:16] = half[:16] if dtype is np.float32 else half[:16].astype(np.float16)
    rows[16:20] = 0.0
    rows[20:24] *= 1e-5
    rows[24:28] *= 6e-8
    rows[28, :, :, ::32] = 60000.0
    rows[29] = np.sign(rows[29]) * 65504.0
    # fp16 halves that fp16 rows can hold: multiples of 0.5 under a largest of 127
    rows[30] = rng.integers(-200, 200, rows[30].shape) * 0.5
    rows[30, ..., ::32] = 127.0
    rows[31, ..., 1:] = 0.0
    if dtype is np.float32:
        rows[32] *= 1e-30
        rows[33] *= 1e-42
        rows[34] = np.sign(rows[34]) * Q.MOST
        rows[35] *= 1e6
    rows = rows.astype(dtype)
    cache, at, got = run(lstk, dev, rng, rows, cells_of(rng, n, 4, "row13"), 4)
    check_back(lstk, dev, cache, at, got)
    if dtype is np.float32:
        back = lstk.load_q8(cache, at, dtype=__import__("torch").float32)[0].cpu().numpy()
        assert np.array_equal(back[34], rows[34, 0])


def test_blocks_that_do_not_fit_hold_nan(lstk, dev):
    """NaN, infinities, and magnitudes above 127 * 65504: that block of 32 dims reads back as NaN, its neighbours as they are."""
    import torch
    rng = np.random.default_rng(6)
    for dtype, bad in ((np.float32, (np.nan, np.inf, -np.inf, 3e38, np.nextafter(np.float32(Q.MOST), np.float32(np.inf)), -1e7)),
                       (np.float16, (np.nan, np.inf, -np.inf))):
        rows = rows_of(rng, len(bad), 2, 64, dtype)
        for i, b in enumerate(bad):
            rows[i, :, 1, 5 + i] = b
        cache, at, got = run(lstk, dev, rng, rows, np.arange(len(bad)) + 3, 2)
        k, v = lstk.load_q8(cache, at, dtype=torch.float32)
        for x in (k, v):
            assert torch.isnan(x[:, 1, :32]).all() and torch.isfinite(x[:, 0]).all() and torch.isfinite(x[:, 1, 32:]).all()


def test_cells_outside_are_left_alone(lstk, dev):
    """Padded rows: cells below 0 and behind the cache write nothing and read as zeros; the others are as without them."""
    rng = np.random.default_rng(7)
    cells = cells_of(rng, 70, 4, "row13")
    cells[[0, 9, 33, 34, 69]] = (-1, 128, 2 ** 31 - 1, -2 ** 31, 129)
    cache, at, got = run(lstk, dev, rng, rows_of(rng, 70, 3, 64, np.float16), cells, 4)
    check_back(lstk, dev, cache, at, got)


def test_strided_rows(lstk, dev):
    """Rows inside wider ones, rows of one tensor for all cells, and outputs inside wider tensors whose other bytes stay."""
    import torch
    rng = np.random.default_rng(8)
    kv, hd, n = 2, 64, 50
    wide = torch.from_numpy(rng.standard_normal((n, 40 + 2 * kv * hd)).astype(np.float32)).to(dev)
    k = wide[:, 8:8 + kv * hd].unflatten(1, (kv, hd))
    v = wide[:, 24 + kv * hd:24 + 2 * kv * hd].unflatten(1, (kv, hd))
    at = torch.arange(5, 5 + n, dtype=torch.int32, device=dev)
    shape = lstk.q8_cache_shape(60, kv, hd)
    assert shape == (2, kv, 68 * hd)
    a, b = (torch.zeros(shape, dtype=torch.uint8, device=dev) for _ in range(2))
    lstk.store_q8(a, k, v, at)
    lstk.store_q8(b, k.contiguous(), v.contiguous(), at)
    assert torch.equal(a, b)
    out = torch.full((n, 3, kv, hd), 7.0, device=dev)
    lstk.load_q8(a, at, k=out[:, 0], v=out[:, 2])
    k2, v2 = lstk.load_q8(a, at, dtype=torch.float32)
    assert torch.equal(out[:, 0], k2) and torch.equal(out[:, 2], v2) and (out[:, 1] == 7.0).all()
    lstk.store_q8(b, k[:1].expand(n, kv, hd), v[:1].expand(n, kv, hd), at)  # one row for all cells
    k3, _ = lstk.load_q8(b, at)
    assert torch.equal(k3, k3[:1].expand_as(k3)) and torch.equal(k3[0], lstk.load_q8(a, at[:1])[0][0])


def test_no_rows(lstk, dev):
    import torch
    cache = torch.full(lstk.q8_cache_shape(32, 2, 64), 3, dtype=torch.uint8, device=dev)
    none = torch.zeros(0, 2, 64, dtype=torch.float16, device=dev)
    at = torch.zeros(0, dtype=torch.int32, device=dev)
    lstk.store_q8(cache, none, none, at)
    assert lstk.load_q8(cache, at)[0].shape == (0, 2, 64) and (cache == 3).all()


def test_captured_and_on_another_stream(lstk, dev):
    """A captured write and read replays over new rows and cells, with eager calls between."""
    import torch
    rng = np.random.default_rng(9)
    kv, hd, n, pages = 2, 128, 40, 6
    rows = torch.from_numpy(rows_of(rng, n, kv, hd, np.float16)).to(dev)
    at = torch.arange(n, dtype=torch.int32, device=dev)
    cache = torch.zeros(pages, kv, 68 * hd, dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    lstk.store_q8(cache, rows[:, 0], rows[:, 1], at, stream=side)
    a = lstk.load_q8(cache, at, stream=side)
    side.synchronize()
    lstk.store_q8(cache, rows[:, 0], rows[:, 1], at)
    assert all(torch.equal(x, y) for x, y in zip(a, lstk.load_q8(cache, at)))
    k, v = torch.zeros(n, kv, hd, dtype=torch.float16, device=dev), torch.zeros(n, kv, hd, dtype=torch.float16, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lstk.store_q8(cache, rows[:, 0], rows[:, 1], at)
        lstk.load_q8(cache, at, k=k, v=v)
    for step in range(4):
        rows.copy_(torch.from_numpy(rows_of(rng, n, kv, hd, np.float16)))
        at.copy_(torch.from_numpy(cells_of(rng, n, pages, ("any", "row7", "back", "row13")[step]).astype(np.int32)))
        g.replay()
        other = torch.zeros_like(cache)
        lstk.store_q8(other, rows[:, 0], rows[:, 1], at)
        k2, v2 = lstk.load_q8(other, at)
        assert torch.equal(k, k2) and torch.equal(v, v2), step


def test_cache_past_32_bit_offsets(lstk, dev):
    """Pages behind 2^32 bytes."""
    import torch
    kv, hd, pages = 8, 256, 40000
    assert pages * kv * 68 * hd > 2 ** 32
    rng = np.random.default_rng(10)
    cache = torch.zeros(pages, kv, 68 * hd, dtype=torch.uint8, device=dev)
    rows = rows_of(rng, 40, kv, hd, np.float16)
    cells = np.concatenate([32 * pages - 1 - np.arange(20), 32 * 31000 + np.arange(20)])
    r = torch.from_numpy(rows).to(dev)
    at = torch.tensor(cells, dtype=torch.int32, device=dev)
    lstk.store_q8(cache, r[:, 0], r[:, 1], at)
    for x, back in zip((rows[:, 0], rows[:, 1]), lstk.load_q8(cache, at, dtype=torch.float32)):
        assert np.array_equal(back.cpu().numpy(), Q.values(*Q.quantise(x)).astype(np.float32))
    assert int((cache != 0).any(2).any(1).sum()) == 2


def test_refusals_of_tensors(lstk, dev):
    import torch
    cache = torch.zeros(lstk.q8_cache_shape(64, 2, 64), dtype=torch.uint8, device=dev)
    x = torch.zeros(5, 2, 64, dtype=torch.float16, device=dev)
    at = torch.arange(5, dtype=torch.int32, device=dev)
    ok = dict(cache=cache, k=x, v=x, cells=at)
    lstk.store_q8(**ok)
    bad = [dict(cache=cache.float()), dict(cache=cache[:, :, :-1].contiguous()), dict(cache=cache.cpu()), dict(cache=cache[:, :, :68 * 32].contiguous()),
           dict(k=x.float()), dict(v=x.float()), dict(k=x.double(), v=x.double()), dict(k=x[:4]), dict(k=x[:, :1]), dict(k=x.cpu()),
           dict(k=x.transpose(1, 2).contiguous().transpose(1, 2)), dict(cells=at.long()), dict(cells=at[:4]), dict(cells=at.cpu()), dict(k=None),
           dict(k=torch.zeros(5 * 132 + 4, dtype=torch.float16, device=dev)[4:].view(5, 132)[:, :128].unflatten(1, (2, 64))),
           dict(cache=torch.zeros(2, 2, 68 * 96, dtype=torch.uint8, device=dev), k=torch.zeros(5, 2, 96, dtype=torch.float16, device=dev),
                v=torch.zeros(5, 2, 96, dtype=torch.float16, device=dev))]
    for b in bad:
        with pytest.raises(lstk.LstkError) as e:
            lstk.store_q8(**{**ok, **b})
        assert e.value.code == lstk.E_INVALID, b
    for b in (dict(dtype=torch.bfloat16), dict(k=x[:1].expand(5, 2, 64)), dict(v=x[:4]), dict(k=x, dtype=torch.float32)):
        with pytest.raises(lstk.LstkError) as e:
            lstk.load_q8(cache, at, **b)
        assert e.value.code == lstk.E_INVALID, b
