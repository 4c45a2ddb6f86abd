"""Attention of one new token per sequence over the paged cache (lstk_attn_paged) against the formula in 64 bits.

Tolerance, per output value, from the kernel's arithmetic (u16 = 2^-11 and u32 = 2^-24, half a step of fp16 and fp32 relative
to the value): a score is a sum of head_dim products rounded to fp32, so it is off by at most E = (head_dim + 4) u32
sum_d |q_d k_d| scale; a weight is off by that, by the exponential (2 u32, and as much again as its argument's rounding, |s| u32)
and by its rounding to fp16 (u16, or 2^-25 of the largest weight where it is a subnormal fp16); the sums over n cells by
(n + 64) u32; the result's own rounding by u16. The weights' errors enter through sum p |v| and, by the division, through |out|.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U16, U32 = 2.0 ** -11, 2.0 ** -24


def make(torch, dev, rng, H, kv, hd, lens, spread=2.0, spare=5, kv_size=None, share=False):
    """Caches in the model's layouts with NaN in every cell that no sequence holds, and the sequences' tables (pages in any
    order, each sequence's list at its own place of the table)."""
    pages = [-(-n // 32) for n in lens]
    total = sum(pages) + spare if kv_size is None else kv_size // 32
    order = rng.permutation(total)[:sum(pages)].astype(np.int32)
    size = total * 32
    K = rng.standard_normal((kv, size, hd)).astype(np.float16)
    V = rng.standard_normal((kv, size, hd)).astype(np.float16)
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
    K[:, ~held] = np.nan
    V[:, ~held] = np.nan
    q = (spread * rng.standard_normal((len(lens), H, hd))).astype(np.float16)
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    kc = d(K.reshape(kv, size, hd // 4, 4).transpose(0, 2, 1, 3))
    vc = d(V.reshape(kv, size // 4, 4, hd).transpose(0, 1, 3, 2))
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
    return dict(K=K, V=V, q=q, rows=rows, kc=kc, vc=vc, qd=d(q), lens=i32(lens), first=i32(first),
                blocks=i32(table if table else [0]), max_len=max(lens + [0]) if lens else 0)


def formula(q, K, V, cells, scale):
    """(out, tolerance) of one sequence's heads over the given cells."""
    H, hd = q.shape
    kv = K.shape[0]
    out, tol = np.zeros((H, hd)), np.full((H, hd), 2.0 ** -24)
    if len(cells) == 0:
        return out, np.zeros((H, hd))
    for h in range(H):
        g = h // (H // kv)
        k, v, x = K[g, cells].astype(np.float64), V[g, cells].astype(np.float64), q[h].astype(np.float64)
        s = k @ x * scale
        e = (hd + 4) * U32 * (np.abs(k) @ np.abs(x)) * abs(scale)
        p = np.exp(s - s.max())
        dp = p * (e + e[np.argmax(s)] + 2 * U32 + np.abs(s - s.max()) * 2 * U32 + U16) + 2.0 ** -25
        t = p.sum()
        o = p @ v / t
        out[h] = o
        a = np.abs(v)
        n = len(cells)
        tol[h] += (dp @ a + np.abs(o) * dp.sum()) / t + 2 * (n + 64) * U32 * (p @ a) / t + U16 * np.abs(o)
    return out, tol


def check(lstk, c, scale=None, window=0, n_sink=0, visible=None, **kw):
    hd = c["q"].shape[2]
    got = lstk.paged_attention(c["qd"], c["kc"], c["vc"], c["lens"], c["first"], c["blocks"], c["max_len"], window=window,
                               n_sink=n_sink, scale=scale, **kw)
    got = got.float().cpu().numpy().astype(np.float64)
    for b, cells in enumerate(c["rows"]):
        n = len(cells)
        i = np.arange(n)
        see = np.ones(n, bool) if window <= 0 else (i >= n - window) | (i < n_sink)
        if visible is not None:
            see &= visible[b]
        want, tol = formula(c["q"][b], c["K"], c["V"], cells[see], hd ** -0.5 if scale is None else scale)
        err = np.abs(got[b] - want)
        assert np.isfinite(got[b]).all(), (b, n)
        assert (err <= tol).all(), (b, n, float((err - tol).max()), float(err.max()))
    return got


HEADS = [(32, 4, 128), (64, 4, 128), (4, 2, 64), (16, 2, 256), (3, 3, 64), (40, 2, 128), (17, 1, 64)]


@pytest.mark.parametrize("H,kv,hd", HEADS)
def test_lengths(lstk, dev, H, kv, hd):
    """Every length around pages, wavefronts and chunks, ragged in one call; empty sequences among them."""
    import torch
    rng = np.random.default_rng(H * hd)
    check(lstk, make(torch, dev, rng, H, kv, hd, [1, 0, 31, 32, 33, 64, 65, 127, 128, 129, 0, 513, 1, 1055, 200]))


@pytest.mark.parametrize("n", [1, 5, 1023, 1024, 1025, 5000, 20011])
def test_one_sequence(lstk, dev, n):
    import torch
    check(lstk, make(torch, dev, np.random.default_rng(n), 32, 4, 128, [n]))


@pytest.mark.parametrize("H,kv,hd", [(32, 4, 128), (4, 2, 64)])
def test_long(lstk, dev, H, kv, hd):
    import torch
    c = make(torch, dev, np.random.default_rng(3), H, kv, hd, [131072, 7, 60001])
    a = check(lstk, c)
    assert np.array_equal(a, check(lstk, c))  # the same bits again


@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 33), (64, 0), (100, 128), (1000, 4), (7, 500), (4096, 4)])
def test_window_and_sinks(lstk, dev, window, n_sink):
    import torch
    rng = np.random.default_rng(window * 7 + n_sink)
    check(lstk, make(torch, dev, rng, 32, 4, 128, [1, 0, 30, 64, 97, 1000, 1024, 1111, 3001]), window=window, n_sink=n_sink)


def test_window_at_every_place_of_a_page(lstk, dev):
    import torch
    rng = np.random.default_rng(5)
    check(lstk, make(torch, dev, rng, 4, 2, 64, list(range(150, 190))), window=65, n_sink=3)


def test_large_scores(lstk, dev):
    """Scores hundreds apart: the maximum moves from page to page, all but a few weights vanish."""
    import torch
    rng = np.random.default_rng(8)
    check(lstk, make(torch, dev, rng, 32, 4, 128, [700, 2000], spread=60.0))
    check(lstk, make(torch, dev, rng, 32, 4, 128, [700, 2000], spread=2.0), scale=-3.0)
    check(lstk, make(torch, dev, rng, 32, 4, 128, [700, 2000]), scale=0.0)


def test_rising_scores(lstk, dev):
    """Each page's scores above the last one's, and the other way round."""
    import torch
    for sign in (1, -1):
        c = make(torch, dev, np.random.default_rng(9), 8, 1, 64, [3000])
        cells = c["rows"][0]
        c["K"][0, cells, 0] = (sign * np.linspace(-40, 40, len(cells))).astype(np.float16)
        c["q"][:, :, 0] = 8.0
        c["kc"].copy_(torch.from_numpy(c["K"].reshape(1, -1, 16, 4).transpose(0, 2, 1, 3).copy()))
        c["qd"].copy_(torch.from_numpy(c["q"]))
        check(lstk, c)


def test_shared_pages(lstk, dev):
    """Sequences that hold the same pages (a shared prompt), of different lengths."""
    import torch
    check(lstk, make(torch, dev, np.random.default_rng(11), 32, 4, 128, [900, 900, 450, 33], share=True))


def test_many_sequences(lstk, dev):
    import torch
    rng = np.random.default_rng(12)
    check(lstk, make(torch, dev, rng, 4, 2, 64, rng.integers(0, 200, 300).tolist()))


@pytest.mark.parametrize("n,longest", [(300, 5000), (257, 3000), (1000, 2500)])
def test_many_sequences_beside_a_long_one(lstk, dev, n, longest):
    """More sequences than a work-group looks up at once, in equal shares of the list of pages."""
    import torch
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 90, n).tolist()
    lens[n // 2], lens[-1], lens[0] = longest, 2100, 0
    c = make(torch, dev, rng, 4, 2, 64, lens)
    assert lstk.paged_attention_work_bytes(n, 4, 2, 64, longest) > 0
    check(lstk, c)
    check(lstk, c, window=1000, n_sink=3)


def test_pages_out_of_range_are_not_visible(lstk, dev):
    """Block numbers outside the cache, and table indices outside the table, hide their cells."""
    import torch
    c = make(torch, dev, np.random.default_rng(13), 32, 4, 128, [400, 200, 40, 70])
    t, first = c["blocks"].cpu().numpy(), c["first"].cpu().numpy()
    size = c["K"].shape[1]
    vis = [np.ones(len(r), bool) for r in c["rows"]]
    for b, p, bad in ((0, 3, -1), (0, 12, size // 32), (1, 0, 2 ** 31 - 1), (2, 0, -2 ** 31), (2, 1, size // 32 + 7)):
        t[first[b] + p] = bad
        vis[b][32 * p:32 * p + 32] = False
    c["blocks"].copy_(torch.from_numpy(t))
    check(lstk, c, visible=vis)  # sequence 2 has no page left: zeros
    # a table that ends inside sequence 3, and a list that starts before it
    c["blocks"] = c["blocks"][:first[3] + 1].contiguous()
    vis[3][32:] = False
    f = first.copy()
    check(lstk, c, visible=vis)
    f[1] = -3
    c["first"].copy_(torch.from_numpy(f))
    vis[1][:96] = False
    cells = (np.maximum(t[:4], 0)[:, None].astype(np.int64) * 32 + np.arange(32)).ravel()
    c["rows"][1] = np.concatenate([np.zeros(96, np.int64), cells])[:200]
    vis[1][96:192] = True
    vis[1][192:] = False  # table entry 3 is one of the bad ones above
    check(lstk, c, visible=vis)


def test_lengths_out_of_range(lstk, dev):
    """A length above max_len counts as max_len, one below zero as zero."""
    import torch
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
    """cell_seq / seqs hide cells that are not the sequence's: some of a page, whole pages, all of a sequence."""
    import torch
    rng = np.random.default_rng(15)
    c = make(torch, dev, rng, 32, 4, 128, [300, 95, 64])
    owner = np.full(c["K"].shape[1], -1, np.int32)
    vis = []
    for b, r in enumerate(c["rows"]):
        keep = rng.random(len(r)) < 0.7
        keep[:40] = False
        if b == 2:
            keep[:] = False
        owner[r[keep]] = 10 + b
        vis.append(keep)
        c["K"][:, r[~keep]] = np.inf
        c["V"][:, r[~keep]] = np.nan
    kv, size, hd = c["K"].shape
    c["kc"].copy_(torch.from_numpy(c["K"].reshape(kv, size, hd // 4, 4).transpose(0, 2, 1, 3).copy()))
    c["vc"].copy_(torch.from_numpy(c["V"].reshape(kv, size // 4, 4, hd).transpose(0, 1, 3, 2).copy()))
    d = lambda a: torch.from_numpy(a).to(dev)
    check(lstk, c, visible=vis, cell_seq=d(owner), seqs=torch.tensor([10, 11, 12], dtype=torch.int32, device=dev))


def test_nan_and_inf_in_view_come_out(lstk, dev):
    """A NaN or an infinite score among the visible cells of a head makes that head's output NaN, and no other sequence's."""
    import torch
    c = make(torch, dev, np.random.default_rng(16), 32, 4, 128, [200, 200])
    for what in (np.nan, np.inf):
        K = c["K"].copy()
        K[1, c["rows"][0][77], 5] = what
        kv, size, hd = K.shape
        kc = torch.from_numpy(K.reshape(kv, size, hd // 4, 4).transpose(0, 2, 1, 3).copy()).to(dev)
        q = c["qd"].abs()
        out = lstk.paged_attention(q, kc, c["vc"], c["lens"], c["first"], c["blocks"], 200).cpu().numpy()
        assert np.isnan(out[0, 8:16]).all() and np.isfinite(out[0, :8]).all() and np.isfinite(out[0, 16:]).all()
        assert np.isfinite(out[1]).all()


def test_rows_behind_stay(lstk, dev):
    """out beyond the last sequence, and the workspace beyond its size, keep what they hold."""
    import torch
    c = make(torch, dev, np.random.default_rng(17), 32, 4, 128, [3000, 100])
    need = lstk.paged_attention_work_bytes(2, 32, 4, 128, 3000)
    assert need > 0
    big, work = torch.full((4, 32, 128), 7.0, dtype=torch.float16, device=dev), torch.full((need + 256,), 9, dtype=torch.uint8, device=dev)
    ref = lstk.paged_attention(c["qd"], c["kc"], c["vc"], c["lens"], c["first"], c["blocks"], 3000)
    L, P = lstk.lib(), lstk.PagedCache
    cache = P(c["kc"].data_ptr(), c["vc"].data_ptr(), c["K"].shape[1], 4, 128, None)
    s = lstk.PagedSeqs(2, 3000, c["lens"].data_ptr(), c["first"].data_ptr(), c["blocks"].data_ptr(), c["blocks"].numel(), None)
    import ctypes
    st = torch.cuda.current_stream().cuda_stream
    assert L.lstk_attn_paged(ctypes.byref(cache), ctypes.byref(s), c["qd"].data_ptr(), 32, 0, 0, 128 ** -0.5, big.data_ptr(),
                             work.data_ptr(), need, st) == 0
    assert torch.equal(big[:2], ref) and (big[2:] == 7.0).all() and (work[need:] == 9).all()


def test_streams_and_capture(lstk, dev):
    """On a stream of its own, and captured: two graphs with a workspace each, replayed several times over changing lengths
    and queries with eager calls between, give the eager results bit for bit."""
    import torch
    c = make(torch, dev, np.random.default_rng(18), 32, 4, 128, [4000, 2500, 64])
    args = lambda s: (s["qd"], s["kc"], s["vc"], s["lens"], s["first"], s["blocks"], 4000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = lstk.paged_attention(*args(c), stream=side)
    side.synchronize()
    check(lstk, c)
    assert torch.equal(a, lstk.paged_attention(*args(c)))
    graphs = []
    for window in (0, 100):
        work = torch.empty(lstk.paged_attention_work_bytes(3, 32, 4, 128, 4000, window, 4), dtype=torch.uint8, device=dev)
        out = torch.zeros_like(c["qd"])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lstk.paged_attention(*args(c), window=window, n_sink=4, out=out, work=work)
        graphs.append((window, g, out, work))
    for step in range(4):
        c["lens"].copy_(torch.tensor([4000 - 700 * step, 2500 - step, step], dtype=torch.int32))
        c["qd"].mul_(0.9)
        for _, g, _, _ in graphs:
            g.replay()
        for window, _, out, _ in graphs:
            ref = lstk.paged_attention(*args(c), window=window, n_sink=4)
            assert torch.equal(out, ref), (step, window)


def test_cache_past_32_bit_offsets(lstk, dev):
    """A cache of more than 2^32 bytes a tensor: pages at its end are read right."""
    import torch
    kv, hd, size = 4, 256, 32 * 70000
    assert kv * hd * size * 2 > 2 ** 32
    kc = torch.zeros(kv, hd // 4, size, 4, dtype=torch.float16, device=dev)
    vc = torch.zeros(kv, size // 4, hd, 4, dtype=torch.float16, device=dev)
    rng = np.random.default_rng(19)
    lens = [100, 70]
    blocks = [69999, 5, 69997, 69998, 40000, 2, 69996]
    first = [0, 4]
    q = (2 * rng.standard_normal((2, 8, hd))).astype(np.float16)
    K, V = {}, {}
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    for b in blocks:
        K[b], V[b] = (rng.standard_normal((kv, 32, hd)).astype(np.float16) for _ in range(2))
        kc[:, :, 32 * b:32 * b + 32] = d(K[b].reshape(kv, 32, hd // 4, 4).transpose(0, 2, 1, 3))
        vc[:, 8 * b:8 * b + 8] = d(V[b].reshape(kv, 8, 4, hd).transpose(0, 1, 3, 2))
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
    got = lstk.paged_attention(d(q), kc, vc, i32(lens), i32(first), i32(blocks), 100).float().cpu().numpy()
    for r in range(2):
        mine = blocks[first[r]:first[r] + -(-lens[r] // 32)]
        k, v = (np.concatenate([x[b] for b in mine], 1) for x in (K, V))
        want, tol = formula(q[r], k, v, np.arange(lens[r]), hd ** -0.5)
        assert (np.abs(got[r] - want) <= tol).all()


def test_refusals_of_tensors(lstk, dev):
    import torch
    c = make(torch, dev, np.random.default_rng(20), 4, 2, 64, [50, 60])
    ok = dict(q=c["qd"], k_cache=c["kc"], v_cache=c["vc"], lens=c["lens"], first=c["first"], blocks=c["blocks"], max_len=60)
    lstk.paged_attention(**ok)
    bad = [dict(q=c["qd"].float()), dict(q=c["qd"].cpu()), dict(q=c["qd"][:, :3].contiguous()), dict(q=c["qd"].transpose(0, 1)),
           dict(k_cache=c["kc"].float()), dict(v_cache=c["kc"]), dict(lens=c["lens"].long()), dict(lens=c["lens"][:1]),
           dict(first=c["first"].cpu()), dict(blocks=c["blocks"].float()), dict(max_len=-1), dict(n_sink=-1), dict(scale=float("nan")),
           dict(scale=float("inf")), dict(out=torch.empty(2, 4, 64, device=dev)), dict(work=torch.empty(8, dtype=torch.uint8)),
           dict(cell_seq=torch.zeros(c["K"].shape[1], dtype=torch.int32, device=dev)), dict(seqs=c["lens"])]
    for b in bad:
        with pytest.raises(lstk.LstkError) as e:
            lstk.paged_attention(**{**ok, **b})
        assert e.value.code == lstk.E_INVALID, b
    with pytest.raises(lstk.LstkError):  # too small a workspace
        lstk.paged_attention(**{**ok, "max_len": 100000, "work": torch.empty(16, dtype=torch.uint8, device=dev)})
    empty = lstk.paged_attention(c["qd"][:0], c["kc"], c["vc"], c["lens"][:0], c["first"][:0], c["blocks"], 60)
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("n_sink", [0, 5])
def test_the_longest_length(lstk, dev, n_sink):
    """A sequence of 2^31 - 1 cells whose window's two pages are the only ones in the table (its list starts before it)."""
    import torch
    c = make(torch, dev, np.random.default_rng(18), 32, 4, 128, [64, 64])
    n, window = 2 ** 31 - 1, 40
    c["max_len"] = n
    c["lens"].fill_(n)
    c["first"].copy_(torch.tensor([2 * b - (2 ** 26 - 2) for b in range(2)], dtype=torch.int32))
    c["rows"] = [r[:63] for r in c["rows"]]  # the second page's last cell would be the one after
    vis = [np.arange(63) >= 63 - window for _ in range(2)]
    check(lstk, c, visible=vis, window=window, n_sink=n_sink)
