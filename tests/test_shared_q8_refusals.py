"""What lstk_cache_q8_store / _load, lstk_attn_paged_q8, lstk_attn_shared(_q8) and lstk_token_logprobs refuse before any device call, and the
sizes of their workspaces (host arithmetic; no GPU)."""
import ctypes

import pytest

P = 4096  # a pointer that no refused call follows
BIG = 2 ** 31 - 1


def rows(lstk, load, **kw):
    a = dict(pages=P, n_pages=2, kv=2, hd=64, k=P, v=P, type=lstk.TYPE_F16, ld_k=128, ld_v=128, cells=P, n=3)
    a.update(kw)
    c = lstk.Q8Cache(a["pages"], a["n_pages"], a["kv"], a["hd"], None)
    f = lstk.lib().lstk_cache_q8_load if load else lstk.lib().lstk_cache_q8_store
    return f(ctypes.byref(c), a["k"], a["v"], a["type"], a["ld_k"], a["ld_v"], a["cells"], a["n"], None)


@pytest.mark.parametrize("load", [False, True])
@pytest.mark.parametrize("kw", [dict(pages=None), dict(pages=P + 8), dict(n_pages=0), dict(n_pages=-1), dict(n_pages=2 ** 22 + 1), dict(kv=0), dict(kv=-2),
                                dict(kv=65536), dict(hd=96), dict(hd=0), dict(hd=512), dict(k=None), dict(k=P + 8), dict(v=None), dict(v=P + 2),
                                dict(type=8), dict(type=-1), dict(ld_k=-8), dict(ld_v=-128), dict(ld_k=132), dict(ld_v=129), dict(cells=None),
                                dict(cells=P + 2), dict(n=-1), dict(n=2 ** 24 + 1), dict(n=2 ** 24, kv=65535)])
def test_cache_rows_refuse(lstk, load, kw):
    assert rows(lstk, load, **kw) == lstk.E_INVALID
    assert lstk.lib().lstk_last_error()


def test_cache_rows(lstk):
    """Rows that are written must not overlap; none at all need no pointers."""
    assert rows(lstk, True, ld_k=64) == rows(lstk, True, ld_v=0) == lstk.E_INVALID
    for load in (False, True):
        assert rows(lstk, load, n=0, k=None, v=None, cells=None, pages=None) == 0
        assert rows(lstk, load, n=0, hd=100) == lstk.E_INVALID
    f = lstk.lib()
    assert f.lstk_cache_q8_store(None, P, P, 1, 128, 128, P, 1, None) == lstk.E_INVALID
    assert lstk.q8_cache_shape(0, 2, 64) == (0, 2, 4352) and lstk.q8_cache_shape(33, 4, 128) == (2, 4, 8704)


def seqs(lstk, a):
    return lstk.PagedSeqs(a["n_seq"], a["max_len"], a["lens"], a["first"], a["blocks"], a["n_table"], a["seq"])


OWN = dict(pages=P, n_pages=2, k=P, v=P, kv_size=64, kv=2, hd=64, cell_seq=None, n_seq=1, max_len=64, lens=P, first=P, blocks=P, n_table=2, seq=None,
           q=P, n_head=4, scale=1.0, out=P, work=None, work_bytes=0)


def attn_q8(lstk, **kw):
    a = {**OWN, "window": 0, "n_sink": 0, **kw}
    c = lstk.Q8Cache(a["pages"], a["n_pages"], a["kv"], a["hd"], a["cell_seq"])
    return lstk.lib().lstk_attn_paged_q8(ctypes.byref(c), ctypes.byref(seqs(lstk, a)), a["q"], a["n_head"], a["window"], a["n_sink"], a["scale"],
                                         a["out"], a["work"], a["work_bytes"], None)


BAD = [dict(q=None), dict(q=P + 8), dict(out=None), dict(out=P + 4), dict(lens=None), dict(lens=P + 2), dict(first=None), dict(first=P + 1),
       dict(blocks=None), dict(blocks=P + 2), dict(hd=96), dict(hd=0), dict(kv=0), dict(kv=3), dict(kv=-2), dict(n_head=0), dict(n_head=-4),
       dict(n_seq=-1), dict(max_len=-1), dict(n_table=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(seq=P), dict(cell_seq=P),
       dict(seq=P + 2, cell_seq=P), dict(kv=65536, n_head=65536), dict(n_seq=BIG, max_len=BIG, work=P, work_bytes=2 ** 62),
       dict(max_len=2 ** 30, work=None, work_bytes=2 ** 40), dict(max_len=2 ** 30, work=P + 8, work_bytes=2 ** 40), dict(max_len=2 ** 30, work=P, work_bytes=64)]


@pytest.mark.parametrize("kw", BAD + [dict(pages=None), dict(pages=P + 8), dict(n_pages=0), dict(n_pages=2 ** 22 + 1), dict(n_sink=-1)])
def test_attention_q8_refuses(lstk, kw):
    assert attn_q8(lstk, **kw) == lstk.E_INVALID
    assert lstk.lib().lstk_last_error()


def shared(lstk, q8, **kw):
    a = {**OWN, "pk": P, "pv": P, "p_size": 64, "p_kv": None, "p_hd": None, "p_seq": None, "p_max": 64, "p_len": P, "p_blocks": P, "p_table": 2, "work": P,
         "work_bytes": 2 ** 40, **kw}
    pc = lstk.PagedCache(a["pk"], a["pv"], a["p_size"], a["p_kv"] or a["kv"], a["p_hd"] or a["hd"], a["p_seq"])
    x = lstk.Prefix(ctypes.pointer(pc), a["p_max"], a["p_len"], a["p_blocks"], a["p_table"])
    c = lstk.Q8Cache(a["pages"], a["n_pages"], a["kv"], a["hd"], a["cell_seq"]) if q8 else \
        lstk.PagedCache(a["k"], a["v"], a["kv_size"], a["kv"], a["hd"], a["cell_seq"])
    f = lstk.lib().lstk_attn_shared_q8 if q8 else lstk.lib().lstk_attn_shared
    return f(ctypes.byref(x), ctypes.byref(c), ctypes.byref(seqs(lstk, a)), a["q"], a["n_head"], a["scale"], a["out"], a["work"], a["work_bytes"], None)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("kw", BAD + [dict(pk=None), dict(pk=P + 8), dict(pv=None), dict(p_size=0), dict(p_size=33), dict(p_size=2 ** 28), dict(p_kv=1),
                                      dict(p_hd=128), dict(p_seq=P), dict(p_max=-1), dict(p_len=None), dict(p_len=P + 2), dict(p_blocks=None),
                                      dict(p_blocks=P + 1), dict(p_table=-1), dict(work=None), dict(work=P + 8), dict(work_bytes=100),
                                      dict(n_seq=2 ** 22 - 1, kv=1, n_head=16, work_bytes=2 ** 62)])
def test_shared_attention_refuses(lstk, q8, kw):
    assert shared(lstk, q8, **kw) == lstk.E_INVALID
    assert lstk.lib().lstk_last_error()


def test_shared_attention_of_one_kind_only(lstk):
    for q8 in (False, True):
        for kw in ((dict(pages=None), dict(n_pages=0), dict(pages=P + 1)) if q8 else (dict(k=None), dict(v=P + 2), dict(kv_size=33))):
            assert shared(lstk, q8, **kw) == lstk.E_INVALID
        assert shared(lstk, q8, n_seq=0, q=None, out=None, lens=None, p_len=None, work=None, work_bytes=0) == 0
    L = lstk.lib()
    x = lstk.Prefix(None, 64, P, P, 2)
    assert L.lstk_attn_shared(None, None, None, P, 4, 1.0, P, None, 0, None) == lstk.E_INVALID
    assert L.lstk_attn_shared(ctypes.byref(x), None, None, P, 4, 1.0, P, None, 0, None) == lstk.E_INVALID


def test_shared_workspace(lstk):
    """More room is never needed for shorter sequences or prefixes; no prefix needs what attention without one needs."""
    w, own = lstk.shared_attention_work_bytes, lstk.paged_attention_q8_work_bytes
    for n, H, kv, hd in ((1, 32, 4, 128), (3, 64, 4, 128), (100, 4, 2, 64), (128, 32, 4, 128), (1000, 16, 2, 256), (7, 40, 2, 128)):
        assert w(n, H, kv, hd, 1, 0) == 0 and w(n, H, kv, hd, 9000, 0) == own(n, H, kv, hd, 9000)
        sizes = [w(n, H, kv, hd, 100, m) for m in list(range(1, 5000, 37)) + [10 ** 4, 10 ** 5, 10 ** 6, BIG]]
        assert sizes == sorted(sizes) and sizes[0] >= n * H * (hd + 4) * 4
        assert sizes[-1] <= max(2 * n, 16384) * H * (hd + 4) * 4
        sizes = [w(n, H, kv, hd, m, 5000) for m in (0, 100, 1000, 10 ** 5, BIG)]
        assert sizes == sorted(sizes)
    assert w(1, 33, 4, 128, 100, 100) == w(1, 32, 4, 100, 100, 100) == w(1, 32, 4, 128, 100, -1) == w(-1, 32, 4, 128, 1, 1) == 0


def logp(lstk, **kw):
    a = dict(x=P, ld=100, n=2, V=100, tok=P, top=2, lp=P, ent=None, ids=P, at=P, work=P, bytes=2 ** 40)
    a.update(kw)
    return lstk.lib().lstk_token_logprobs(a["x"], a["ld"], a["n"], a["V"], a["tok"], a["top"], a["lp"], a["ent"], a["ids"], a["at"], a["work"], a["bytes"],
                                          None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(x=P + 2), dict(ld=99), dict(n=-1), dict(V=0), dict(V=-1), dict(V=2 ** 20 - 15, ld=2 ** 20), dict(tok=None),
                                dict(tok=P + 1), dict(top=-1), dict(top=33), dict(lp=None), dict(lp=P + 2), dict(ent=P + 2), dict(ids=None),
                                dict(ids=P + 2), dict(at=None), dict(at=P + 1), dict(n=2 ** 22, V=100), dict(V=50000, ld=50000, work=None),
                                dict(V=50000, ld=50000, work=P + 8), dict(V=50000, ld=50000, bytes=100)])
def test_logprobs_refuse(lstk, kw):
    assert logp(lstk, **kw) == lstk.E_INVALID
    assert lstk.lib().lstk_last_error()


def test_logprobs_workspace(lstk):
    assert logp(lstk, n=0, x=None, tok=None, lp=None, ids=None, at=None, work=None, bytes=0) == 0
    w = lstk.token_logprobs_work_bytes
    assert w(0, 100) == w(1, 0) == w(1, 2 ** 20 - 15) == w(1, 100, 33) == w(1, 100, -1) == w(5, 2000, 4) == 0
    assert 0 < w(1, 151936) < w(1, 151936, 20) < w(64, 151936, 20) < 2 ** 20
    assert w(1, 2 ** 20 - 16, 32) == 64 * (16 + 8 * 32)


def test_tensors_on_the_host_are_refused(lstk):
    torch = pytest.importorskip("torch")
    x, cache = torch.zeros(2, 16), torch.zeros(2, 2, 68 * 64, dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    r = torch.zeros(2, 2, 64, dtype=torch.float16)
    k = torch.zeros(2, 16, 64, 4, dtype=torch.float16)
    for f in (lambda: lstk.token_logprobs(x, i), lambda: lstk.store_q8(cache, r, r, i), lambda: lstk.load_q8(cache, i),
              lambda: lstk.paged_attention_q8(q, cache, i, i, i, 5), lambda: lstk.SharedPrefix(k, k, i[:1], i, 5),
              lambda: lstk.shared_attention(q, None, k, k, i, i, i, 5), lambda: lstk.token_logprobs(None, i), lambda: lstk.store_q8(None, r, r, i)):
        with pytest.raises(lstk.LstkError) as e:
            f()
        assert e.value.code == lstk.E_INVALID
