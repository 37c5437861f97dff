"""Queries keep all bits of a float32 number over pages of every type."""
import numpy as np
import pytest

from test_gpu_paged import TYPES, _ctx, _ints, hip, torch  # noqa: F401

pytestmark = pytest.mark.gpu

P = 16


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [8, 64, 96, 128, 256])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -3, 2.0 ** 2])
def test_queries_of_24_bits(hip, torch, size, hd, dtype):  # noqa: F811
    """Two queries' numbers that differ in their last bit against a key that subtracts them: products with 1 and the one sum are exact in
    float32, so the score is that bit, and with values 1 and -1 the output is tanh of half of it."""
    H = 4
    ctx = _ctx(hip, torch, H, 1, hd)
    cache = hip.PagedKVCache(ctx, 2, P, 1, 2, dtype=dtype)
    cache.table.copy_(_ints(torch, [[1, 0]]))
    big = 2.0 ** 14
    # key 0: big, -big in two places; key 1: nothing
    cache.k[1, 0, 0, 1], cache.k[1, 0, 0, hd - 2] = big, -big
    cache.v[1, 0, 0], cache.v[1, 0, 1] = 1.0, -1.0
    last = np.array([1.0, 3.0, -1.0, 2.0 ** 8 + 1]) * 2.0 ** -23
    q = np.zeros((H, hd), np.float32)
    q[:, 1] = size * (1 + 2.0 ** -12 + last)
    q[:, hd - 2] = size * (1 + 2.0 ** -12)
    out = ctx.attend_paged(cache, _ints(torch, [0]), _ints(torch, [1]), torch.from_numpy(q.reshape(1, -1)).cuda())
    ctx.sync()
    want = np.tanh(size * last * big / np.sqrt(hd) / 2)
    # weights near 1/2, their sum and its quotient: a few half steps of 1
    assert np.abs(out.cpu().numpy().reshape(H, hd) - want[:, None]).max() <= 16 * 2.0 ** -24 + 4 * 2.0 ** -24 * np.abs(want).max()
