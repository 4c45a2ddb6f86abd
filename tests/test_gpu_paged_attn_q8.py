"""Attention of one new token per sequence over the cache in 8 bits (lstk_attn_paged_q8) against the formula in 64 bits on the values d q.

Tolerance, per output value, from the kernel's arithmetic (u16 = 2^-11, u32 = 2^-24: half a step relative to the value). A score is a
sum of head_dim exact products in blocks of 32, each block's sum rounded to fp32 step by step, then times its scale and added up: off by
at most E = (head_dim + 12) u32 sum_d |q_d k_d| scale. A weight p is off by that, by the exponential and its argument's rounding (2 u32 and
2 |s| u32), by its product with the scale of V (u32), and by that product's two fp16 parts: 2^-22 of it, or 2^-25 where the second part is
a subnormal number. The largest p is at least 2^15 over twice the largest scale, so 2^-25 of a product with a scale d is at most
2^-39 d_max / d of the largest weight (2^-38 below). The sums over n cells by (n + 64) u32; the result's own rounding by u16 (2^-25 if it
is subnormal).
"""
import numpy as np
import pytest

import q8_cache as Q

pytestmark = pytest.mark.gpu

U16, U32 = 2.0 ** -11, 2.0 ** -24


def make(torch, dev, rng, H, kv, hd, lens, spread=2.0, spare=5, share=False, large=1.0):
    """A cache whose cells that no sequence holds have NaN scales and any bytes, and the sequences' tables."""
    pages = [-(-n // 32) for n in lens]
    total = sum(pages) + spare
    order = rng.permutation(total)[:sum(pages)].astype(np.int32)
    size = total * 32
    parts = []
    for _ in range(2):
        d, q = Q.quantise((rng.standard_normal((kv, size, hd)) * np.where(np.arange(hd) % 32 == 3, large, 1.0)).astype(np.float32))
        parts += [d, q]
    first, table, at, rows = [], [], 0, []
    held = np.zeros(size, bool)
    for n, p in zip(lens, pages):
        first.append(len(table))
        blk = order[at:at + p] if not (share and rows) else order[:p]
        at += 0 if share and rows else p
        table += blk.tolist()
        cells = (blk[:, None].astype(np.int64) * 32 + np.arange(32)).ravel()[:n]
        held[cells] = True
        rows.append(cells)
    for i in (0, 2):
        parts[i][:, ~held] = np.where(rng.random((kv, int((~held).sum()), hd // 32)) < 0.5, np.float16(np.nan), np.float16(np.inf))
        parts[i + 1][:, ~held] = rng.integers(-128, 128, parts[i + 1][:, ~held].shape)
    q = (spread * rng.standard_normal((len(lens), H, hd))).astype(np.float16)
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
    with np.errstate(invalid="ignore"):
        K, V = Q.values(*parts[:2]), Q.values(*parts[2:])
    return dict(K=K, V=V, kd=parts[0], vd=parts[2], parts=parts, q=q, rows=rows, cache=d(Q.pack(*parts)), qd=d(q), lens=i32(lens),
                first=i32(first), blocks=i32(table if table else [0]), max_len=max(lens + [0]) if lens else 0)


def formula(q, K, V, vd, cells, scale):
    """(out, tolerance) of one sequence's heads over the given cells."""
    H, hd = q.shape
    kv = K.shape[0]
    out, tol = np.zeros((H, hd)), np.full((H, hd), 2.0 ** -25)
    if len(cells) == 0:
        return out, np.zeros((H, hd))
    for h in range(H):
        g = h // (H // kv)
        k, v, x = K[g, cells], V[g, cells], q[h].astype(np.float64)
        s = k @ x * scale
        e = (hd + 12) * U32 * (np.abs(k) @ np.abs(x)) * abs(scale)
        p = np.exp(s - s.max())
        scales = vd[g, cells].astype(np.float64)
        small = scales[scales > 0]
        spread = small.max() / small.min() if small.size else 1.0
        dp = p * (e + e[np.argmax(s)] + 4 * U32 + np.abs(s - s.max()) * 2 * U32 + 2.0 ** -22) + spread * 2.0 ** -38
        t = p.sum()
        o = p @ v / t
        out[h] = o
        n = len(cells)
        tol[h] += (dp @ np.abs(v) + np.abs(o) * dp.sum()) / t + 2 * (n + 64) * U32 * (p @ np.abs(v)) / t + U16 * np.abs(o)
    return out, tol


def check(lstk, c, scale=None, window=0, n_sink=0, visible=None, **kw):
    hd = c["q"].shape[2]
    got = lstk.paged_attention_q8(c["qd"], c["cache"], c["lens"], c["first"], c["blocks"], c["max_len"], window=window, n_sink=n_sink,
                                  scale=scale, **kw)
    got = got.float().cpu().numpy().astype(np.float64)
    for b, cells in enumerate(c["rows"]):
        n = len(cells)
        i = np.arange(n)
        see = np.ones(n, bool) if window <= 0 else (i >= n - window) | (i < n_sink)
        if visible is not None:
            see &= visible[b]
        want, tol = formula(c["q"][b], c["K"], c["V"], c["vd"], cells[see], hd ** -0.5 if scale is None else scale)
        err = np.abs(got[b] - want)
        assert np.isfinite(got[b]).all(), (b, n)
        assert (err <= tol).all(), (b, n, float((err - tol).max()), float(err.max()))
    return got


HEADS = [(32, 4, 128), (64, 4, 128), (4, 2, 64), (16, 2, 256), (3, 3, 64), (40, 2, 128), (17, 1, 64)]


@pytest.mark.parametrize("H,kv,hd", HEADS)
def test_lengths(lstk, dev, H, kv, hd):
    import torch
    rng = np.random.default_rng(H * hd)
    check(lstk, make(torch, dev, rng, H, kv, hd, [1, 0, 31, 32, 33, 64, 65, 127, 128, 129, 0, 513, 1, 1055, 200]))


@pytest.mark.parametrize("n", [1, 5, 1023, 1024, 1025, 5000, 20011])
def test_one_sequence(lstk, dev, n):
    import torch
    check(lstk, make(torch, dev, np.random.default_rng(n), 32, 4, 128, [n]))


@pytest.mark.parametrize("H,kv,hd", [(32, 4, 128), (4, 2, 64), (16, 2, 256)])
def test_long(lstk, dev, H, kv, hd):
    import torch
    c = make(torch, dev, np.random.default_rng(3), H, kv, hd, [70000, 7, 30001])
    a = check(lstk, c)
    assert np.array_equal(a, check(lstk, c))  # the same bits again


@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 33), (100, 128), (1000, 4), (7, 500), (4096, 4)])
def test_window_and_sinks(lstk, dev, window, n_sink):
    import torch
    rng = np.random.default_rng(window * 7 + n_sink)
    check(lstk, make(torch, dev, rng, 32, 4, 128, [1, 0, 30, 64, 97, 1000, 1024, 1111, 3001]), window=window, n_sink=n_sink)


def test_large_and_rising_scores(lstk, dev):
    import torch
    rng = np.random.default_rng(8)
    check(lstk, make(torch, dev, rng, 32, 4, 128, [700, 2000], spread=60.0))
    check(lstk, make(torch, dev, rng, 32, 4, 128, [700, 2000]), scale=-3.0)
    check(lstk, make(torch, dev, rng, 32, 4, 128, [700, 2000]), scale=0.0)


@pytest.mark.parametrize("large", [30.0, 1000.0, 1e-3])
def test_blocks_with_one_large_dim(lstk, dev, large):
    import torch
    check(lstk, make(torch, dev, np.random.default_rng(9), 16, 4, 128, [600, 45], large=large))


@pytest.mark.parametrize("by", [2.0 ** -14, 2.0 ** -7, 2.0 ** 9, 2.0 ** 13])
def test_scales_at_the_ends_of_fp16(lstk, dev, by):
    """Scales of V from 2^-21 (subnormal fp16 numbers) to 2^8: weights times scales stay inside fp16 and keep their bits."""
    import torch
    c = make(torch, dev, np.random.default_rng(10), 8, 2, 64, [300, 33])
    vd, vq = c["parts"][2], c["parts"][3]
    for cells in c["rows"]:
        vd[:, cells] = (vd[:, cells].astype(np.float64) * by).astype(np.float16)
    c["V"] = Q.values(vd, vq)
    c["cache"].copy_(torch.from_numpy(Q.pack(*c["parts"])))
    check(lstk, c)


def test_a_hundred_thousand_small_weights(lstk, dev):
    """One cell 20 above all others in units of log 2, the others' weights add up to a tenth of it: none of them is lost."""
    import torch
    n, hd = 100000, 64
    c = make(torch, dev, np.random.default_rng(11), 2, 1, hd, [n])
    kd, kq, vd, vq = c["parts"]
    cells = c["rows"][0]
    kd[0, cells] = np.float16(1.0)
    kq[0, cells] = 0
    kq[0, cells[77], 0, 0] = 64
    vd[0, cells] = np.float16(0.5)
    vq[0, cells] = 100
    vq[0, cells[77]] = -100
    c["q"][:] = 0
    c["q"][:, :, 0] = 1.0
    c["K"], c["V"] = Q.values(kd, kq), Q.values(vd, vq)
    c["cache"].copy_(torch.from_numpy(Q.pack(*c["parts"])))
    c["qd"].copy_(torch.from_numpy(c["q"]))
    check(lstk, c, scale=20.0 * np.log(2.0) / 64.0)


def test_pages_out_of_range_and_lengths(lstk, dev):
    import torch
    c = make(torch, dev, np.random.default_rng(13), 32, 4, 128, [400, 200, 40, 70])
    t, first = c["blocks"].cpu().numpy(), c["first"].cpu().numpy()
    pages = c["cache"].shape[0]
    vis = [np.ones(len(r), bool) for r in c["rows"]]
    for b, p, bad in ((0, 3, -1), (0, 12, pages), (1, 0, 2 ** 31 - 1), (2, 0, -2 ** 31), (2, 1, pages + 7)):
        t[first[b] + p] = bad
        vis[b][32 * p:32 * p + 32] = False
    c["blocks"].copy_(torch.from_numpy(t))
    check(lstk, c, visible=vis)
    c["blocks"] = c["blocks"][:first[3] + 1].contiguous()
    vis[3][32:] = False
    check(lstk, c, visible=vis)
    c = make(torch, dev, np.random.default_rng(14), 32, 4, 128, [500, 40])
    c["max_len"] = 333
    c["rows"][0] = c["rows"][0][:333]
    check(lstk, c)
    c["lens"].copy_(torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32))
    c["rows"][1] = c["rows"][1][:0]
    check(lstk, c)
    c["max_len"] = 0
    c["rows"][0] = c["rows"][0][:0]
    assert not check(lstk, c).any()


def test_cells_of_other_owners(lstk, dev):
    import torch
    rng = np.random.default_rng(15)
    c = make(torch, dev, rng, 32, 4, 128, [300, 95, 64])
    owner = np.full(32 * c["cache"].shape[0], -1, np.int32)
    vis = []
    for b, r in enumerate(c["rows"]):
        keep = rng.random(len(r)) < 0.7
        keep[:40] = False
        if b == 2:
            keep[:] = False
        owner[r[keep]] = 10 + b
        vis.append(keep)
        c["parts"][0][:, r[~keep]] = np.inf
        c["parts"][2][:, r[~keep]] = np.nan
    c["cache"].copy_(torch.from_numpy(Q.pack(*c["parts"])))
    check(lstk, c, visible=vis, cell_seq=torch.from_numpy(owner).to(dev), seqs=torch.tensor([10, 11, 12], dtype=torch.int32, device=dev))


def test_nan_in_view_comes_out(lstk, dev):
    """A block of K that holds NaN makes its heads' outputs NaN, one of V those dims, and no other sequence's."""
    import torch
    c = make(torch, dev, np.random.default_rng(16), 32, 4, 128, [200, 200])
    for i in (0, 2):
        parts = [p.copy() for p in c["parts"]]
        parts[i][1, c["rows"][0][77], 2] = np.nan
        cache = torch.from_numpy(Q.pack(*parts)).to(dev)
        out = lstk.paged_attention_q8(c["qd"], cache, c["lens"], c["first"], c["blocks"], 200).cpu().numpy()
        bad = out[0, 8:16] if i == 0 else out[0, 8:16, 64:96]
        assert np.isnan(bad).all() and np.isfinite(out[0, :8]).all() and np.isfinite(out[0, 16:]).all() and np.isfinite(out[1]).all()


@pytest.mark.parametrize("n,longest", [(300, 5000), (257, 3000)])
def test_many_sequences_beside_a_long_one(lstk, dev, n, longest):
    import torch
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 90, n).tolist()
    lens[n // 2], lens[-1], lens[0] = longest, 2100, 0
    c = make(torch, dev, rng, 4, 2, 64, lens)
    check(lstk, c)
    check(lstk, c, window=1000, n_sink=3)


def test_shared_pages_of_stored_rows(lstk, dev):
    """Rows that store_q8 wrote, read through lists that share pages: the attention of what load_q8 gives back."""
    import torch
    rng = np.random.default_rng(17)
    c = make(torch, dev, rng, 32, 4, 128, [900, 900, 450, 33], share=True)
    rows = rng.standard_normal((900, 2, 4, 128)).astype(np.float32)
    cells = torch.tensor(c["rows"][0], dtype=torch.int32, device=dev)
    r = torch.from_numpy(rows).to(dev)
    lstk.store_q8(c["cache"], r[:, 0], r[:, 1], cells)
    k, v = lstk.load_q8(c["cache"], cells, dtype=torch.float32)
    c["K"][:, c["rows"][0]], c["V"][:, c["rows"][0]] = (x.double().cpu().numpy().transpose(1, 0, 2) for x in (k, v))
    c["vd"] = Q.unpack(c["cache"].cpu().numpy())[2]
    check(lstk, c)


def test_rows_behind_stay_and_graphs(lstk, dev):
    """out beyond the last sequence and the workspace beyond its size keep what they hold; two graphs with a workspace each replay over
    changing lengths and queries, with eager calls between, and give the eager results bit for bit."""
    import torch
    c = make(torch, dev, np.random.default_rng(18), 32, 4, 128, [4000, 2500, 64])
    args = lambda: (c["qd"], c["cache"], c["lens"], c["first"], c["blocks"], 4000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = lstk.paged_attention_q8(*args(), stream=side)
    side.synchronize()
    assert torch.equal(a, lstk.paged_attention_q8(*args()))
    need = lstk.paged_attention_q8_work_bytes(3, 32, 4, 128, 4000)
    big, work = torch.full((5, 32, 128), 7.0, dtype=torch.float16, device=dev), torch.full((need + 256,), 9, dtype=torch.uint8, device=dev)
    lstk.paged_attention_q8(*args(), out=big[:3], work=work[:need])
    assert torch.equal(big[:3], a) and (big[3:] == 7.0).all() and (work[need:] == 9).all()
    graphs = []
    for window in (0, 100):
        work = torch.empty(lstk.paged_attention_q8_work_bytes(3, 32, 4, 128, 4000, window, 4), dtype=torch.uint8, device=dev)
        out = torch.zeros_like(c["qd"])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lstk.paged_attention_q8(*args(), window=window, n_sink=4, out=out, work=work)
        graphs.append((window, g, out, work))
    for step in range(4):
        c["lens"].copy_(torch.tensor([4000 - 700 * step, 2500 - step, step], dtype=torch.int32))
        c["qd"].mul_(0.9)
        for _, g, _, _ in graphs:
            g.replay()
        for window, _, out, _ in graphs:
            assert torch.equal(out, lstk.paged_attention_q8(*args(), window=window, n_sink=4)), (step, window)


def test_refusals_of_tensors(lstk, dev):
    import torch
    c = make(torch, dev, np.random.default_rng(20), 4, 2, 64, [50, 60])
    ok = dict(q=c["qd"], cache=c["cache"], lens=c["lens"], first=c["first"], blocks=c["blocks"], max_len=60)
    lstk.paged_attention_q8(**ok)
    bad = [dict(q=c["qd"].float()), dict(q=c["qd"].cpu()), dict(q=c["qd"][:, :3].contiguous()), dict(q=c["qd"][..., :32].contiguous()),
           dict(cache=c["cache"].float()), dict(cache=c["cache"][:, :, 1:].contiguous()), dict(lens=c["lens"].long()), dict(lens=c["lens"][:1]),
           dict(first=c["first"].cpu()), dict(blocks=c["blocks"].float()), dict(max_len=-1), dict(n_sink=-1), dict(scale=float("nan")),
           dict(max_len=2 ** 31), dict(window=2 ** 31), dict(out=torch.empty(2, 4, 64, device=dev)), dict(work=torch.empty(8, dtype=torch.uint8)),
           dict(cell_seq=torch.zeros(32 * c["cache"].shape[0], dtype=torch.int32, device=dev)), dict(seqs=c["lens"])]
    for b in bad:
        with pytest.raises(lstk.LstkError) as e:
            lstk.paged_attention_q8(**{**ok, **b})
        assert e.value.code == lstk.E_INVALID, b
    with pytest.raises(lstk.LstkError):
        lstk.paged_attention_q8(**{**ok, "max_len": 100000, "work": torch.empty(16, dtype=torch.uint8, device=dev)})
    assert lstk.paged_attention_q8(c["qd"][:0], c["cache"], c["lens"][:0], c["first"][:0], c["blocks"], 60).shape == (0, 4, 64)
