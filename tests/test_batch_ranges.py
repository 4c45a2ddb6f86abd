"""Numbers that 32-bit arguments cannot hold are refused, not cut to their lower bits (no GPU: every call ends before the library's,
or the library refuses it)."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

BIG = [2 ** 32, 2 ** 32 + 7, 2 ** 32 + 64, 2 ** 31, -2 ** 31 - 1, -2 ** 32 + 5, 2 ** 80]


def refused(lstk, what, f):
    with pytest.raises(lstk.LstkError) as e:
        f()
    assert e.value.code == lstk.E_INVALID and what in str(e.value), str(e.value)


@pytest.fixture
def calls(lstk, monkeypatch):
    """Stands in for a GPU: tensors of the host pass the checks of tensors, and library calls are counted instead of made."""
    made = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: made.append(name) or 0
    monkeypatch.setattr(lstk, "lib", Lib)
    monkeypatch.setattr(lstk, "_on_device", lambda dev, stream, call: call(None))
    monkeypatch.setattr(lstk, "_tensor", lambda t, name, dtype, shape, dev=None: t.data_ptr())
    monkeypatch.setattr(lstk, "_rows", lambda t, name, dtype: (t.data_ptr(), t.shape[1], *t.shape, -1))
    monkeypatch.setattr(lstk, "_empty", lambda shape, dtype, dev, stream: torch.empty(shape, dtype=dtype))
    return made


def attention(lstk, **kw):
    h = dict(dtype=torch.float16)
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    a = dict(q=torch.zeros(1, 4, 64, **h), k_cache=torch.zeros(2, 16, 64, 4, **h), v_cache=torch.zeros(2, 16, 64, 4, **h), lens=i(7), first=i(0),
             blocks=i(0, 1), max_len=64, work=torch.zeros(64))
    return lstk.paged_attention(**{**a, **kw})


@pytest.mark.parametrize("v", BIG)
@pytest.mark.parametrize("name", ["max_len", "window", "n_sink"])
def test_attention(lstk, calls, name, v):
    refused(lstk, name, lambda: attention(lstk, **{name: v}))
    assert not calls
    attention(lstk)
    attention(lstk, max_len=2 ** 31 - 1, window=-1)
    assert calls == ["lstk_attn_paged"] * 2


@pytest.mark.parametrize("v", BIG)
def test_workspaces(lstk, v):
    for i, name in enumerate(("n_seq", "n_head", "n_head_kv", "head_dim", "max_len", "window", "n_sink")):
        a = [1, 4, 2, 64, 64, 0, 0]
        a[i] = v
        refused(lstk, name, lambda: lstk.paged_attention_work_bytes(*a))
    refused(lstk, "n_rows", lambda: lstk.sample_work_bytes(v, 100))
    refused(lstk, "n_vocab", lambda: lstk.sample_work_bytes(1, v))


@pytest.mark.parametrize("v", BIG)
def test_rules(lstk, calls, v):
    for name in ("n_group", "n_group_used", "group_top"):
        refused(lstk, name, lambda: lstk.RouterRule(**{name: v}))
    refused(lstk, "n_expert_used", lambda: lstk.moe_select(torch.zeros(0, 16), v, lstk.RouterRule()))
    assert not calls


@pytest.mark.parametrize("v", BIG)
def test_batch_steps(lstk, v):
    m = lstk.Qwen3Model.__new__(lstk.Qwen3Model)
    m.hp, m._h, m.n_batch, m.device, m.logits = dict(n_layer=2, n_vocab=16, n_expert_used=2), None, 4, torch.device("cpu"), torch.zeros(16)
    for name in ("window", "n_sink"):
        refused(lstk, name, lambda: m.decode_batch([0], [1], logits=4096, **{name: v}))
        refused(lstk, name, lambda: m.forward_batch(1, 10, logits=4096, **{name: v}))
    refused(lstk, "max_len", lambda: m.forward_batch(1, v, logits=4096))
    refused(lstk, "n_seq", lambda: m.forward_batch(v, 10, logits=4096))
    as_given = [[v], np.array([v], dtype=object)] + ([np.array([v], np.int64), torch.tensor([v])] if abs(v) < 2 ** 63 else [])
    for a in as_given:
        for f in (m.decode_batch, m.prepare_batch):
            refused(lstk, "sequences", lambda: f(a, [1]))
            refused(lstk, "tokens", lambda: f([1], a))
    store = lstk.ExpertStore(1, 256, 512, 8, 2, 4, [((8, 8, 8), None, None, None)], dry=True)
    for name in ("layer", "gate_type", "n_tokens"):
        a = dict(dict(layer=0, gate_type=1, n_tokens=1), **{name: v})
        refused(lstk, name, lambda: store.route_by(rule=lstk.RouterRule(), hnorm=4096, gate_inp=4096, ids=4096, weights=4096, **a))


def test_ids_of_every_kind(lstk):
    for a in ([1, 2], (1, 2), range(1, 3), np.array([1, 2]), np.array([1.0, 2.0]), np.array([[1], [2]], np.uint8), torch.tensor([1, 2])):
        got = lstk._ids32(a, "x")
        assert got.dtype == np.int32 and got.tolist() == [1, 2] and got.flags.c_contiguous
    assert lstk._ids32([], "x").size == 0
    for a in ([1.5], [float("nan")], [float("inf")], ["a"], [None], np.array([3e9]), [[1], [2, 3]], iter([1])):
        with pytest.raises(lstk.LstkError):
            lstk._ids32(a, "x")
