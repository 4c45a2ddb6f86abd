"""What lstk_attn_paged, lstk_sample, lstk_moe_select and the batch step refuse before any device call, and the sizes of their
workspaces (host arithmetic; no GPU)."""
import ctypes

import pytest

P = 4096  # a pointer that no refused call follows


def attn(lstk, **kw):
    a = dict(k=P, v=P, kv_size=64, n_kv=2, hd=64, cell_seq=None, n_seq=1, max_len=64, lens=P, first=P, blocks=P, n_table=2, seq=None, q=P,
             n_head=4, window=0, n_sink=0, scale=1.0, out=P, work=None, work_bytes=0)
    a.update(kw)
    c = lstk.PagedCache(a["k"], a["v"], a["kv_size"], a["n_kv"], a["hd"], a["cell_seq"])
    s = lstk.PagedSeqs(a["n_seq"], a["max_len"], a["lens"], a["first"], a["blocks"], a["n_table"], a["seq"])
    return lstk.lib().lstk_attn_paged(ctypes.byref(c), ctypes.byref(s), a["q"], a["n_head"], a["window"], a["n_sink"], a["scale"], a["out"],
                                      a["work"], a["work_bytes"], None)


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 2), dict(q=None), dict(q=P + 8), dict(out=None), dict(out=P + 4),
                                dict(lens=None), dict(lens=P + 2), dict(first=None), dict(first=P + 1), dict(blocks=None), dict(blocks=P + 2),
                                dict(kv_size=0), dict(kv_size=33), dict(kv_size=-32), dict(kv_size=2 ** 31), dict(hd=96), dict(hd=0), dict(hd=512),
                                dict(n_kv=0), dict(n_kv=3), dict(n_kv=-2), dict(n_head=0), dict(n_head=-4), dict(n_seq=-1), dict(max_len=-1),
                                dict(n_sink=-1), dict(n_table=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(seq=P), dict(cell_seq=P),
                                dict(seq=P + 2, cell_seq=P), dict(max_len=2 ** 30, work=P, work_bytes=64), dict(max_len=2 ** 30, work=None, work_bytes=2 ** 40),
                                dict(max_len=2 ** 30, work=P + 8, work_bytes=2 ** 40), dict(n_seq=2 ** 31 - 1, max_len=2 ** 31 - 1, work=P, work_bytes=2 ** 62),
                                dict(n_kv=65536, n_head=65536)])
def test_attention_refuses(lstk, kw):
    assert attn(lstk, **kw) == lstk.E_INVALID
    assert lstk.lib().lstk_last_error()


def test_attention_of_no_sequences_does_nothing(lstk):
    assert attn(lstk, n_seq=0, q=None, out=None, lens=None) == 0
    assert lstk.lib().lstk_attn_paged(None, None, P, 4, 0, 0, 1.0, P, None, 0, None) == lstk.E_INVALID


def test_attention_workspace(lstk):
    """More room is never needed for shorter sequences; short ones need none; rejected shapes need none."""
    w = lstk.paged_attention_work_bytes
    for n, H, kv, hd in ((1, 32, 4, 128), (3, 64, 4, 128), (100, 4, 2, 64), (1000, 16, 2, 256), (7, 40, 2, 128)):
        assert w(n, H, kv, hd, 1) == w(n, H, kv, hd, 32) == w(n, H, kv, hd, 0) == 0
        sizes = [w(n, H, kv, hd, m) for m in list(range(1, 5000, 37)) + [10 ** 4, 10 ** 5, 10 ** 6, 2 ** 31 - 1]]
        assert sizes == sorted(sizes)
        assert sizes[-1] <= max(n, 4096) * H * (hd + 4) * 4
        assert w(n, H, kv, hd, 10 ** 6, 4096, 4) <= sizes[-1]
    assert w(1, 33, 4, 128, 10 ** 6) == w(1, 32, 4, 100, 10 ** 6) == w(-1, 32, 4, 128, 10 ** 6) == w(1, 32, 0, 128, 10 ** 6) == 0


def sample(lstk, **kw):
    a = dict(x=P, ld=100, n=2, V=100, T=None, k=None, p=None, m=None, u=P, tok=P, prob=None, work=P, bytes=2 ** 40)
    a.update(kw)
    h = lstk.Sampling(a["T"], a["k"], a["p"], a["m"])
    return lstk.lib().lstk_sample(a["x"], a["ld"], a["n"], a["V"], ctypes.byref(h), a["u"], a["tok"], a["prob"], a["work"], a["bytes"], None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(x=P + 2), dict(ld=99), dict(n=-1), dict(V=0), dict(V=-5), dict(V=2 ** 20, ld=2 ** 20), dict(n=2 ** 30, bytes=2 ** 62), dict(u=None),
                                dict(u=P + 1), dict(tok=None), dict(tok=P + 2), dict(prob=P + 2), dict(T=P + 2), dict(k=P + 2), dict(p=P + 1),
                                dict(m=P + 3), dict(work=None), dict(work=P + 4), dict(bytes=100)])
def test_sample_refuses(lstk, kw):
    assert sample(lstk, **kw) == lstk.E_INVALID


def test_sample_workspace(lstk):
    assert sample(lstk, n=0, x=None, u=None, tok=None, work=None) == 0
    assert lstk.sample_work_bytes(0, 100) == lstk.sample_work_bytes(1, 0) == lstk.sample_work_bytes(1, 2 ** 20) == 0
    assert 0 < lstk.sample_work_bytes(1, 1) <= lstk.sample_work_bytes(1, 151936) < lstk.sample_work_bytes(64, 151936) < 2 ** 27
    assert lstk.lib().lstk_sample(P, 100, 1, 100, None, P, P, None, P, 2 ** 40, None) == lstk.E_INVALID


def select(lstk, **kw):
    a = dict(score=0, n_group=1, used=1, top=1, renorm=1, scale=1.0, x=P, ld=16, bias=None, T=2, E=16, k=2, ids=P, w=P)
    a.update(kw)
    r = lstk.CRouterRule(a["score"], a["n_group"], a["used"], a["top"], a["renorm"], a["scale"])
    return lstk.lib().lstk_moe_select(ctypes.byref(r), a["x"], a["ld"], a["bias"], a["T"], a["E"], a["k"], a["ids"], a["w"], None)


@pytest.mark.parametrize("kw", [dict(score=2), dict(score=-1), dict(n_group=0), dict(n_group=3), dict(n_group=4, used=0), dict(n_group=4, used=5),
                                dict(n_group=4, used=-1), dict(n_group=-4), dict(top=0), dict(top=3), dict(n_group=16, used=2, top=2),
                                dict(n_group=8, used=1, k=3), dict(scale=float("nan")), dict(scale=float("inf")), dict(E=0), dict(E=257, ld=257),
                                dict(E=-16), dict(k=0), dict(k=17), dict(k=-1), dict(E=128, ld=128, k=65), dict(T=-1), dict(T=2 ** 24 + 1), dict(ld=15), dict(x=None),
                                dict(x=P + 2), dict(bias=P + 2), dict(ids=None), dict(ids=P + 1), dict(w=None), dict(w=P + 2)])
def test_select_refuses(lstk, kw):
    assert select(lstk, **kw) == lstk.E_INVALID
    assert lstk.lib().lstk_last_error()


def test_select_of_no_tokens_does_nothing(lstk):
    assert select(lstk, T=0, x=None, ids=None, w=None) == 0
    assert lstk.lib().lstk_moe_select(None, P, 16, None, 2, 16, 2, P, P, None) == lstk.E_INVALID
    with pytest.raises(lstk.LstkError):
        lstk.RouterRule("tanh")


def test_batch_entries_refuse_null(lstk):
    L = lstk.lib()
    one = (ctypes.c_int32 * 1)(0)
    n = ctypes.c_int32()
    assert L.lstk_model_decode_batch(None, 1, one, one, 0, 0, P, None, None) == lstk.E_INVALID
    assert L.lstk_model_prepare_batch(None, 1, one, one, ctypes.byref(n), None) == lstk.E_INVALID
    assert L.lstk_model_prepare_batch(P, 1, one, one, None, None) == lstk.E_INVALID
    assert L.lstk_model_forward_batch(None, 1, 1, 0, 0, P, None, None) == lstk.E_INVALID
    assert L.lstk_moe_route_by(None, 0, None, P, 1, P, 1, None, P, P, None) == lstk.E_INVALID


def test_tensors_on_the_host_are_refused(lstk):
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 16)
    for f in (lambda: lstk.moe_select(x, 2, lstk.RouterRule()), lambda: lstk.sample(x, torch.zeros(2)),
              lambda: lstk.paged_attention(torch.zeros(1, 4, 64, dtype=torch.float16), *[None] * 5, 32)):
        with pytest.raises(lstk.LstkError) as e:
            f()
        assert e.value.code == lstk.E_INVALID


def test_a_stream_of_another_gpu_is_refused(lstk):
    """Before the call is made; the stream stands for one of GPU 1, the tensors' is GPU 0."""
    class Other:
        cuda_stream, device_index = P, 1
    called = []
    with pytest.raises(lstk.LstkError) as e:
        lstk._on_device(0, Other(), called.append)
    assert e.value.code == lstk.E_INVALID and not called


def test_attention_counts_tasks_before_it_plans(lstk):
    """Sequences times heads times pages past 2^63: refused, with no workspace, from the number of tasks alone."""
    big = dict(n_seq=2 ** 31 - 1, n_head=65535, n_kv=65535, max_len=2 ** 31 - 1)
    assert attn(lstk, **big, work=P, work_bytes=2 ** 62) == lstk.E_INVALID
    assert b"too many" in lstk.lib().lstk_last_error()
    assert lstk.paged_attention_work_bytes(2 ** 31 - 1, 65535, 65535, 64, 2 ** 31 - 1) == 0
