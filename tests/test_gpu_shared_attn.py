"""Attention over cells that all sequences share and each one's own behind them (lstk_attn_shared, lstk_attn_shared_q8) against the formula
in 64 bits over all of a sequence's cells.

Tolerance: that of attention over the fp16 cache (test_gpu_paged_attn.py), whose weights count one rounding to fp16 (2^-11) as those of
the prefix have it, and 2^-25 of the largest as the least that a weight may be off by (the kernel: half a step of the subnormal numbers,
2^-25, at a largest weight of 2^12 or more). Values of a quantised cache are those that it holds (d q), fp32 products with 8-bit
numbers being no less exact than with fp16 ones.
"""
import numpy as np
import pytest

import q8_cache as Q
from test_gpu_paged_attn import formula, make

pytestmark = pytest.mark.gpu


def build(torch, dev, rng, H, kv, hd, prefix, lens, spread=2.0, bits=16, one_cache=False):
    """A prefix in a cache of its own (or the sequences'), cells that nobody holds full of NaN, and the sequences' own cells."""
    if one_cache:
        c = make(torch, dev, rng, H, kv, hd, lens + [prefix], spread=spread)
        p = dict(K=c["K"], V=c["V"], kc=c["kc"], vc=c["vc"], cells=c["rows"].pop())
        f = int(c["first"][-1])
        p["blocks"] = c["blocks"][f:].contiguous()
        c["lens"], c["first"], c["qd"], c["q"] = c["lens"][:-1].contiguous(), c["first"][:-1].contiguous(), c["qd"][:-1].contiguous(), c["q"][:-1]
    else:
        c = make(torch, dev, rng, H, kv, hd, lens, spread=spread)
        x = make(torch, dev, rng, H, kv, hd, [prefix])
        p = dict(K=x["K"], V=x["V"], kc=x["kc"], vc=x["vc"], cells=x["rows"][0], blocks=x["blocks"])
    c["max_len"] = max(lens + [0])
    if bits == 8:
        size = c["K"].shape[1]
        parts = []
        for a in (c["K"], c["V"]):
            parts += Q.quantise(np.nan_to_num(a).astype(np.float32))
            parts[-2][:, np.isnan(a[0, :, 0])] = np.nan
        c["cache"] = torch.from_numpy(Q.pack(*parts)).to(dev)
        c["K"], c["V"] = Q.values(*parts[:2]), Q.values(*parts[2:])
        assert size == 32 * c["cache"].shape[0]
    p["length"] = torch.tensor([prefix], dtype=torch.int32, device=dev)
    p["max_len"] = prefix
    c["p"] = p
    return c


def call(lstk, c, **kw):
    p = c["p"]
    prefix = lstk.SharedPrefix(p["kc"], p["vc"], p["length"], p["blocks"], p["max_len"])
    s = (c["lens"], c["first"], c["blocks"], c["max_len"])
    if "cache" in c:
        return lstk.shared_attention_q8(c["qd"], prefix, c["cache"], *s, **kw)
    return lstk.shared_attention(c["qd"], prefix, c["kc"], c["vc"], *s, **kw)


def check(lstk, c, scale=None, seen=None, own_seen=None, **kw):
    hd, p = c["q"].shape[2], c["p"]
    got = call(lstk, c, scale=scale, **kw).float().cpu().numpy().astype(np.float64)
    pc = p["cells"] if seen is None else p["cells"][seen]
    for b, cells in enumerate(c["rows"]):
        cells = cells if own_seen is None else cells[own_seen[b]]
        K, V = (np.concatenate([a[:, pc].astype(np.float64), o[:, cells].astype(np.float64)], 1) for a, o in ((p["K"], c["K"]), (p["V"], c["V"])))
        want, tol = formula(c["q"][b], K, V, np.arange(K.shape[1]), hd ** -0.5 if scale is None else scale)
        err = np.abs(got[b] - want)
        assert np.isfinite(got[b]).all(), (b, len(cells))
        assert (err <= tol).all(), (b, len(cells), float((err - tol).max()), float(err.max()))
    return got


HEADS = [(32, 4, 128), (4, 2, 64), (16, 2, 256), (3, 3, 64), (40, 2, 128), (17, 1, 64)]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("H,kv,hd", HEADS)
@pytest.mark.parametrize("prefix", [1, 31, 33, 200, 1055])
def test_lengths(lstk, dev, H, kv, hd, prefix, bits):
    import torch
    rng = np.random.default_rng(H * hd + prefix)
    check(lstk, build(torch, dev, rng, H, kv, hd, prefix, [1, 0, 31, 32, 33, 64, 129, 0, 513, 1], bits=bits))


@pytest.mark.parametrize("H,kv,hd,n", [(32, 4, 128, 1), (32, 4, 128, 8), (32, 4, 128, 9), (32, 4, 128, 16), (32, 4, 128, 17), (16, 1, 64, 33),
                                       (16, 2, 256, 40), (16, 2, 256, 3), (64, 4, 128, 13), (5, 5, 64, 100)])
def test_batches(lstk, dev, H, kv, hd, n):
    """Row blocks that are full, one row more, and few rows, over a prefix of many shares."""
    import torch
    rng = np.random.default_rng(n)
    check(lstk, build(torch, dev, rng, H, kv, hd, 3001, rng.integers(0, 70, n).tolist()))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n,own", [(3, 5000), (40, 900)])
def test_long_own_cells(lstk, dev, n, own, bits):
    """The own cells' pages in equal shares, whose parts meet in a launch of their own."""
    import torch
    rng = np.random.default_rng(own)
    lens = rng.integers(own // 2, own, n).tolist()
    lens[1] = 0
    c = build(torch, dev, rng, 32, 4, 128, 2000, lens, bits=bits)
    a = check(lstk, c)
    assert np.array_equal(a, check(lstk, c))


def test_long_prefix(lstk, dev):
    import torch
    c = build(torch, dev, np.random.default_rng(3), 8, 1, 64, 70001, [5, 0, 40] + [3] * 13)
    a = check(lstk, c)
    assert np.array_equal(a, check(lstk, c))


def test_as_paged_attention_over_lists_that_begin_alike(lstk, dev):
    """One cache for both: what lstk_attn_paged gives when every list begins with the prefix's pages, to the two roundings."""
    import torch
    rng = np.random.default_rng(4)
    c = build(torch, dev, rng, 32, 4, 128, 640, [100, 64, 1, 0, 333], one_cache=True)
    a = check(lstk, c)
    lists, first = [], []
    b, f, n = c["blocks"].cpu().numpy(), c["first"].cpu().numpy(), c["lens"].cpu().numpy()
    for i in range(5):
        first.append(len(lists))
        lists += c["p"]["blocks"].cpu().tolist() + b[f[i]:f[i] + -(-n[i] // 32)].tolist()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    other = lstk.paged_attention(c["qd"], c["kc"], c["vc"], i32(n + 640), i32(first), i32(lists), 973).float().cpu().numpy()
    for i in range(5):
        cells = np.concatenate([c["p"]["cells"], c["rows"][i]])
        _, tol = formula(c["q"][i], c["K"], c["V"], cells, 128 ** -0.5)
        assert (np.abs(a[i] - other[i]) <= 2 * tol).all()


def test_large_and_rising_scores(lstk, dev):
    import torch
    rng = np.random.default_rng(5)
    for n in (3, 40):
        check(lstk, build(torch, dev, rng, 8, 2, 64, 700, [50] * n, spread=60.0))
        check(lstk, build(torch, dev, rng, 8, 2, 64, 700, [50] * n), scale=-3.0)
        check(lstk, build(torch, dev, rng, 8, 2, 64, 77, [50] * n), scale=0.0)
        for sign in (1, -1):
            c = build(torch, dev, rng, 8, 1, 64, 3000, [40] * n)
            p = c["p"]
            p["K"][0, p["cells"], 0] = (sign * np.linspace(-40, 40, 3000)).astype(np.float16)
            c["q"][:, :, 0] = 8.0
            p["kc"].copy_(torch.from_numpy(p["K"].reshape(1, -1, 16, 4).transpose(0, 2, 1, 3).copy()))
            c["qd"].copy_(torch.from_numpy(c["q"]))
            check(lstk, c)


@pytest.mark.parametrize("n", [2, 20])
def test_a_hundred_thousand_small_weights(lstk, dev, n):
    """A cell of the prefix 20 above all others in units of log 2, first or last, the others' weights a tenth of it in all: none is lost."""
    import torch
    for big in (3, 99990):
        c = build(torch, dev, np.random.default_rng(6), 4, 1, 64, 100000, [0, 5] * (n // 2))
        p, cells = c["p"], c["p"]["cells"]
        p["K"][0, cells] = 0
        p["K"][0, cells[big], 0] = 64
        p["V"][0, cells] = 50
        p["V"][0, cells[big]] = -50
        c["q"][:] = 0
        c["q"][:, :, 0] = 1.0
        p["kc"].copy_(torch.from_numpy(p["K"].reshape(1, -1, 16, 4).transpose(0, 2, 1, 3).copy()))
        p["vc"].copy_(torch.from_numpy(p["V"].reshape(1, -1, 4, 64).transpose(0, 1, 3, 2).copy()))
        c["qd"].copy_(torch.from_numpy(c["q"]))
        got = check(lstk, c, scale=20.0 * np.log(2.0) / 64.0)
        w = 99999 * 2.0 ** -20
        assert np.abs(got[0] - 50 * (w - 1) / (w + 1)).max() <= 50 * 2.0 ** -10


@pytest.mark.parametrize("value", [3.0e4, 6.5e4])
def test_huge_scores(lstk, dev, value):
    """Scores of 10^9 and more, where a difference of two is rounded to whole steps: finite outputs, and the cell that is ahead by many
    steps alone decides."""
    import torch
    for n in (2, 20):
        c = build(torch, dev, np.random.default_rng(7), 8, 1, 64, 500, [3] * n)
        c["q"][:] = value
        p = c["p"]
        p["K"][0, p["cells"]] = 100.0
        p["K"][0, p["cells"][300]] = 30000.0
        c["K"][0, :, :] = np.where(np.isnan(c["K"][0]), np.nan, -5.0)
        for k, dst in ((p["K"], p["kc"]), (c["K"], c["kc"])):
            dst.copy_(torch.from_numpy(k.reshape(1, -1, 16, 4).transpose(0, 2, 1, 3).copy()))
        c["qd"].copy_(torch.from_numpy(c["q"]))
        got = call(lstk, c).float().cpu().numpy()
        assert np.array_equal(got, np.broadcast_to(p["V"][0, p["cells"][300]].astype(np.float32), got.shape))


def test_pages_out_of_range_and_lengths(lstk, dev):
    import torch
    for n in (3, 20):
        c = build(torch, dev, np.random.default_rng(8), 32, 4, 128, 400, [30] * n)
        p = c["p"]
        t = p["blocks"].cpu().numpy()
        seen = np.ones(400, bool)
        for j, bad in ((0, -1), (3, p["K"].shape[1] // 32), (5, 2 ** 31 - 1), (12, -2 ** 31)):
            t[j] = bad
            seen[32 * j:32 * j + 32] = False
        p["blocks"].copy_(torch.from_numpy(t))
        check(lstk, c, seen=seen)
        p["blocks"] = p["blocks"][:7].contiguous()  # a table that ends before the prefix
        seen[7 * 32:] = False
        check(lstk, c, seen=seen)
        p["max_len"] = 70  # a length above max_len counts as max_len, one below zero as zero
        seen[70:] = False
        check(lstk, c, seen=seen)
        p["length"].fill_(-7)
        check(lstk, c, seen=seen[:400] & False)
        p["length"].fill_(0)
        check(lstk, c, seen=seen[:400] & False)
        p["max_len"] = 0
        check(lstk, c, seen=seen[:400] & False)


def test_nothing_visible_gives_zeros(lstk, dev):
    import torch
    for n in (2, 20):
        for bits in (16, 8):
            c = build(torch, dev, np.random.default_rng(9), 32, 4, 128, 64, [0, 5] * (n // 2), bits=bits)
            c["p"]["length"].zero_()
            got = check(lstk, c, seen=np.zeros(64, bool))
            assert not got[::2].any() and got[1::2].any()


def test_own_cells_of_other_owners(lstk, dev):
    import torch
    rng = np.random.default_rng(10)
    c = build(torch, dev, rng, 32, 4, 128, 100, [300, 95, 64])
    owner = np.full(c["K"].shape[1], -1, np.int32)
    vis = []
    for b, r in enumerate(c["rows"]):
        keep = rng.random(len(r)) < 0.7
        if b == 2:
            keep[:] = False
        owner[r[keep]] = 10 + b
        vis.append(keep)
    check(lstk, c, own_seen=vis, cell_seq=torch.from_numpy(owner).to(dev), seqs=torch.tensor([10, 11, 12], dtype=torch.int32, device=dev))


def test_nan_in_the_prefix_comes_out(lstk, dev):
    import torch
    for n in (2, 20):
        c = build(torch, dev, np.random.default_rng(11), 32, 4, 128, 200, [5] * n)
        p = c["p"]
        K = p["K"].copy()
        K[1, p["cells"][77], 5] = np.nan
        p["kc"].copy_(torch.from_numpy(K.reshape(4, -1, 32, 4).transpose(0, 2, 1, 3).copy()))
        out = call(lstk, c).cpu().numpy()
        assert np.isnan(out[:, 8:16]).all() and np.isfinite(out[:, :8]).all() and np.isfinite(out[:, 16:]).all()


def test_rows_behind_stay(lstk, dev):
    import torch
    c = build(torch, dev, np.random.default_rng(12), 32, 4, 128, 1500, [900, 0, 30] * 7)
    n = 21
    need = lstk.shared_attention_work_bytes(n, 32, 4, 128, 900, 1500)
    ref = call(lstk, c)
    big, work = torch.full((n + 3, 32, 128), 7.0, dtype=torch.float16, device=dev), torch.full((need + 256,), 9, dtype=torch.uint8, device=dev)
    call(lstk, c, out=big[:n], work=work[:need])
    assert torch.equal(big[:n], ref) and (big[n:] == 7.0).all() and (work[need:] == 9).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_streams_and_capture(lstk, dev, bits):
    """Two graphs with a workspace each, replayed over changing prefixes, lengths and queries with eager calls between."""
    import torch
    cs = [build(torch, dev, np.random.default_rng(13 + i), 32, 4, 128, 1000, [700, 20, 64] * m, bits=bits) for i, m in enumerate((1, 8))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = call(lstk, cs[0], stream=side)
    side.synchronize()
    assert torch.equal(a, call(lstk, cs[0]))
    graphs = []
    for c in cs:
        work = torch.empty(lstk.shared_attention_work_bytes(len(c["rows"]), 32, 4, 128, 700, 1000), dtype=torch.uint8, device=dev)
        out = torch.zeros_like(c["qd"])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(lstk, c, out=out, work=work)
        graphs.append((c, g, out, work))
    for step in range(4):
        for c, g, _, _ in graphs:
            c["p"]["length"].fill_(1000 - 320 * step)
            c["lens"][1] = 20 - step
            c["qd"].mul_(0.9)
            g.replay()
        for c, _, out, _ in graphs:
            assert torch.equal(out, call(lstk, c)), step


def test_refusals_of_tensors(lstk, dev):
    import torch
    c = build(torch, dev, np.random.default_rng(14), 4, 2, 64, 50, [5, 6])
    e = build(torch, dev, np.random.default_rng(14), 4, 2, 64, 50, [5, 6], bits=8)
    other = build(torch, dev, np.random.default_rng(14), 4, 4, 64, 50, [5, 6])["p"]
    wide = build(torch, dev, np.random.default_rng(14), 4, 2, 128, 50, [5, 6])["p"]
    p = c["p"]
    P = lambda x=p, **kw: lstk.SharedPrefix(*{**dict(k=x["kc"], v=x["vc"], n=x["length"], b=x["blocks"], m=x["max_len"]), **kw}.values())
    for kw in (dict(k=p["kc"].float()), dict(k=p["kc"].cpu()), dict(v=p["kc"]), dict(n=p["length"].long()), dict(n=p["length"].cpu()),
               dict(n=torch.zeros(2, dtype=torch.int32, device=dev)), dict(b=p["blocks"].long()), dict(m=2 ** 31), dict(m="x")):
        with pytest.raises(lstk.LstkError) as err:
            P(**kw)
        assert err.value.code == lstk.E_INVALID, kw
    s = (c["lens"], c["first"], c["blocks"], 6)
    lstk.shared_attention(c["qd"], P(), c["kc"], c["vc"], *s)
    lstk.shared_attention_q8(e["qd"], P(), e["cache"], e["lens"], e["first"], e["blocks"], 6)
    calls = [lambda **k: lstk.shared_attention(**{**dict(q=c["qd"], prefix=P(), k_cache=c["kc"], v_cache=c["vc"], lens=s[0], first=s[1], blocks=s[2], max_len=6), **k}),
             lambda **k: lstk.shared_attention_q8(**{**dict(q=e["qd"], prefix=P(), cache=e["cache"], lens=s[0], first=s[1], blocks=s[2], max_len=6), **k})]
    for f in calls:
        f()
        for k in (dict(prefix=None), dict(prefix=P(other)), dict(prefix=P(wide)), dict(prefix=P(m=-1)), dict(q=c["qd"].float()), dict(q=c["qd"][:1]),
                  dict(lens=s[0].long()), dict(max_len=-1), dict(max_len=2 ** 31), dict(scale=float("inf")), dict(out=c["qd"].float()),
                  dict(work=torch.empty(16, dtype=torch.uint8, device=dev)), dict(seqs=s[0]), dict(q=c["qd"][:, :3].contiguous())):
            with pytest.raises(lstk.LstkError) as err:
                f(**k)
            assert err.value.code == lstk.E_INVALID, k
    assert lstk.shared_attention(c["qd"][:0], P(), c["kc"], c["vc"], s[0][:0], s[1][:0], s[2], 6).shape == (0, 4, 64)
