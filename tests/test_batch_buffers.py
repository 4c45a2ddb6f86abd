"""What batch steps and routing by a rule refuse about the buffers they are given, before any device call: host memory, other
types, fewer elements than the kernels read or write."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

HP = dict(n_layer=2, n_embd=256, n_vocab=16, n_expert=8, n_expert_used=2)


def refused(lstk, what, f):
    with pytest.raises(lstk.LstkError) as e:
        f()
    assert e.value.code == lstk.E_INVALID and what in str(e.value), str(e.value)


@pytest.fixture
def model(lstk):
    """A model that was never created on a device: the library would refuse its null handle, so a message that names the buffer
    comes from the look at it."""
    m = lstk.Qwen3Model.__new__(lstk.Qwen3Model)
    m.hp, m._h, m.n_batch, m.device, m.logits = HP, None, 4, torch.device("cpu"), torch.zeros(16)
    return m


CASES = [("logits", torch.zeros(2, 16)), ("logits", np.zeros((2, 16), np.float32)), ("logits", torch.zeros(1, 16)),
         ("logits", torch.zeros(2, 16, dtype=torch.float16)), ("logits", torch.zeros(16, 2).t()), ("logits", 1.5),
         ("trace", torch.zeros(2, 2, 2, dtype=torch.int32)), ("trace", torch.zeros(7, dtype=torch.int32)), ("trace", torch.zeros(2, 2, 2)),
         ("trace", torch.zeros(2, 2, 2, dtype=torch.int64)), ("trace", np.zeros(8, np.int32))]


@pytest.mark.parametrize("name,value", CASES)
def test_batch_steps_look_at_what_they_write(lstk, model, name, value):
    kw = dict({} if name == "logits" else dict(logits=4096), **{name: value})
    refused(lstk, name, lambda: model.decode_batch([0, 1], [1, 2], **kw))
    refused(lstk, name, lambda: model.forward_batch(2, 10, **kw))


def test_raw_pointers_pass(lstk, model, monkeypatch):
    """As everywhere in this module: an integer is a device pointer, None is none."""
    monkeypatch.setattr(lstk, "_on_device", lambda dev, stream, call: call(None))
    for kw in (dict(logits=4096), dict(logits=4096, trace=8192), dict(logits=4096, trace=None)):
        refused(lstk, "null argument", lambda: model.decode_batch([0, 1], [1, 2], **kw))


@pytest.mark.parametrize("name,value", [("bias", torch.zeros(8)), ("bias", torch.zeros(7)), ("bias", torch.zeros(8, dtype=torch.float64)),
                                        ("bias", np.zeros(8, np.float32)), ("ids", torch.zeros(3, 2, dtype=torch.int32)),
                                        ("ids", torch.zeros(3, 2, dtype=torch.int64)), ("ids", torch.zeros(5, dtype=torch.int32)),
                                        ("weights", torch.zeros(3, 2)), ("weights", torch.zeros(3, 2).half()), ("weights", torch.zeros(2, 2)),
                                        ("hnorm", torch.zeros(3, 256)), ("hnorm", torch.zeros(3, 256).half()), ("hnorm", torch.zeros(2, 256)),
                                        ("gate_inp", torch.zeros(8, 256).half()), ("gate_inp", torch.zeros(8, 255).half())])
def test_route_by_looks_at_what_it_reads_and_writes(lstk, name, value):
    store = lstk.ExpertStore(1, 256, 512, 8, 2, 4, [((8, 8, 8), None, None, None)], dry=True)
    a = dict(hnorm=4096, gate_inp=4096, ids=4096, weights=4096, bias=None)
    a[name] = value
    refused(lstk, name, lambda: store.route_by(0, lstk.RouterRule(), gate_type=lstk.TYPE_F16, n_tokens=3, **a))
    refused(lstk, "dry pool", lambda: store.route_by(0, lstk.RouterRule(), 4096, 4096, lstk.TYPE_F16, 4096, 4096, n_tokens=3))


@pytest.mark.gpu
def test_a_model_refuses_them_before_it_appends(lstk, dev):
    from test_gpu_batch_step import build, weights
    hp, w = weights("tiny")
    store, m = build(lstk, dev, hp, w, n_batch=4, kv_size=256)
    m.decode(0, [1, 2, 3])
    z = lambda *s, t=torch.int32, d=dev: torch.zeros(*s, dtype=t, device=d)
    for name, v in (("logits", z(2, 1024, t=torch.float32, d="cpu")), ("trace", z(2, 2, 2, d="cpu")), ("trace", z(7)), ("trace", z(2, 2, 2, t=torch.int64))):
        refused(lstk, name, lambda: m.decode_batch([0, 1], [1, 2], **{name: v}))
        assert (m.seq_len(0), m.seq_len(1)) == (3, 0)
    tr = z(9)
    m.decode_batch([0, 1], [1, 2], trace=tr)
    assert tr[8] == 0 and m.seq_len(1) == 1
    x, gate = z(3, 256, t=torch.float32), z(8, 256, t=torch.float16)
    ids, wts = z(3, 2), z(3, 2, t=torch.float32)
    for bias in (z(7, t=torch.float32), z(8, t=torch.float64), z(8, t=torch.float32, d="cpu")):
        refused(lstk, "bias", lambda: store.route_by(0, lstk.RouterRule(), x, gate, lstk.TYPE_F16, ids, wts, bias=bias))
    store.route_by(0, lstk.RouterRule(), x, gate, lstk.TYPE_F16, ids, wts, bias=z(8, t=torch.float32))
    assert ids.cpu().tolist() == [[0, 1]] * 3
    m.close()
    store.close()
