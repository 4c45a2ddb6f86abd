"""Where what the 8-bit cache holds of fp16 rows lies past fp16's range: by the format in numpy for every fp16 value (no GPU), and what
load_q8 gives there."""
import numpy as np
import pytest

import q8_cache as Q


def ends():
    """Blocks of 32: the largest, a value below it (65504 .. 65184), and zeros."""
    large = [65504.0, 65472.0, 65440.0]
    below = np.arange(65184.0, 65505.0, 32.0)
    rows = [[m, v, -v] + [0.0] * 29 for m in large for v in below if v <= m]
    return np.array(rows, np.float16)


def test_which_values_pass_the_range():
    """A block whose largest is 65440 or less holds nothing past fp16's range; in one of 65472 or 65504 values from 65280 on are held as 65532."""
    x = np.arange(1, 0x7c00, dtype=np.uint16).view(np.float16)
    d, q = Q.quantise(np.pad(x[:, None], ((0, 0), (0, 31))))
    with np.errstate(over="ignore"):
        back = Q.values(d, q)[:, 0].astype(np.float16)
    assert x[np.isinf(back)].tolist() == [65472.0, 65504.0]
    r = ends()
    held = Q.values(*Q.quantise(r))
    passed = (np.abs(r[:, :1]) >= 65472) & (np.abs(r) >= 65280)
    assert (np.abs(held[passed]) == 65532).all() and (np.abs(held[~passed]) < 65520).all()
    assert np.abs(held - r).max() <= 258  # (d / 2)


@pytest.mark.gpu
def test_load(lstk, dev):
    import torch
    r = ends()
    rows = torch.from_numpy(np.tile(r[:, None], (1, 2, 2))).to(dev)  # [n][2][64]
    n = len(r)
    cache = torch.zeros(lstk.q8_cache_shape(n, 2, 64), dtype=torch.uint8, device=dev)
    at = torch.arange(n, dtype=torch.int32, device=dev)
    lstk.store_q8(cache, rows, rows, at)
    held = np.tile(Q.values(*Q.quantise(r))[:, None], (1, 2, 2))
    for x in lstk.load_q8(cache, at, dtype=torch.float32):
        assert np.array_equal(x.cpu().numpy(), held.astype(np.float32))
    for x in lstk.load_q8(cache, at):
        x = x.cpu().numpy()
        passed = np.abs(held) > 65519
        assert np.isinf(x[passed]).all() and np.array_equal(np.signbit(x[passed]), held[passed] < 0)
        assert np.isfinite(x[~passed]).all() and passed.any(1).any(1).sum() < n
