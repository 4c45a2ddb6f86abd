"""Caches whose pages lie behind 2^32 bytes: attention over the 8-bit cache, and over a shared prefix by few and by many sequences."""
import numpy as np
import pytest

import q8_cache as Q
import test_gpu_paged_attn as f16
import test_gpu_paged_attn_q8 as q8

pytestmark = pytest.mark.gpu


def test_the_8_bit_cache(lstk, dev):
    import torch
    kv, hd, pages = 8, 256, 40000
    assert pages * kv * 68 * hd > 2 ** 32
    rng = np.random.default_rng(1)
    cache = torch.full((pages, kv, 68 * hd), 255, dtype=torch.uint8, device=dev)  # scales of NaN
    lens, blocks, first = [100, 70, 33], [39999, 5, 39997, 39998, 20000, 2, 39996, 31000, 31001], [0, 4, 7]
    used = np.unique(blocks)
    parts = []
    for _ in range(2):
        parts += Q.quantise(rng.standard_normal((kv, 32 * len(used), hd)).astype(np.float32))
    cache[torch.from_numpy(used).to(dev)] = torch.from_numpy(Q.pack(*parts)).to(dev)
    where = {int(b): i for i, b in enumerate(used)}
    q = (2 * rng.standard_normal((3, 16, hd))).astype(np.float16)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
    got = lstk.paged_attention_q8(torch.from_numpy(q).to(dev), cache, i32(lens), i32(first), i32(blocks), 100).float().cpu().numpy()
    K, V = Q.values(*parts[:2]), Q.values(*parts[2:])
    for r in range(3):
        cells = np.concatenate([32 * where[b] + np.arange(32) for b in blocks[first[r]:first[r] + -(-lens[r] // 32)]])[:lens[r]]
        want, tol = q8.formula(q[r], K, V, parts[2], cells, hd ** -0.5)
        assert (np.abs(got[r] - want) <= tol).all()


@pytest.mark.parametrize("n", [2, 40])
def test_a_prefix(lstk, dev, n):
    import torch
    kv, hd, size, H = 4, 256, 32 * 70000, 16
    assert kv * hd * size * 2 > 2 ** 32
    rng = np.random.default_rng(2)
    nan = torch.full((), float("nan"), dtype=torch.float16, device=dev)
    kc, vc = nan.expand(kv, hd // 4, size, 4).contiguous(), nan.expand(kv, size // 4, hd, 4).contiguous()
    blocks = [69999, 7, 69990, 40000, 3, 69998, 65536]
    length = 32 * 6 + 5
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    K, V = (rng.standard_normal((kv, 32 * len(blocks), hd)).astype(np.float16) for _ in range(2))
    for i, b in enumerate(blocks):
        k, v = K[:, 32 * i:32 * i + 32], V[:, 32 * i:32 * i + 32]
        kc[:, :, 32 * b:32 * b + 32] = d(k.reshape(kv, 32, hd // 4, 4).transpose(0, 2, 1, 3))
        vc[:, 8 * b:8 * b + 8] = d(v.reshape(kv, 8, 4, hd).transpose(0, 1, 3, 2))
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
    q = (2 * rng.standard_normal((n, H, hd))).astype(np.float16)
    prefix = lstk.SharedPrefix(kc, vc, i32([length]), i32(blocks), length)
    lens = [33 if i % 2 else 0 for i in range(n)]  # own cells: the prefix's pages 0 and 5, in the same cache
    got = lstk.shared_attention(d(q), prefix, kc, vc, i32(lens), i32([0] * n), i32([blocks[0], blocks[5]]), 33).float().cpu().numpy()
    for r in range(n):
        cells = np.concatenate([np.arange(length), np.arange(32), 32 * 5 + np.arange(1)]) if lens[r] else np.arange(length)
        want, tol = f16.formula(q[r], K, V, cells, hd ** -0.5)
        assert (np.abs(got[r] - want) <= tol).all()
