"""A cache in pages without a GPU: the plain model that the GPU tests use, and the calls that are refused on the host."""
import ctypes as C
import os

import numpy as np
import pytest

import shainet_amd
from paged_model import Pages, attended
from shainet_amd import hip


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(shainet_amd.library_path()):
        shainet_amd.build_library(force=False)
    return hip.lib()


def test_plain_pages_come_back_in_order():
    m = Pages(6, 8, 3, 4)
    assert [r[0] for r in m.map([(1, 9), (0, 1)], 20)] == [0, 1, 2, 3, 4, 5, 6, 7, 8, 16]
    before = list(m.free), list(m.lens)
    assert m.map([(1, -2), (2, 20)], 20)[0] == (8, 0, 2)  # the page that sequence 1 gave back
    assert m.map([(1, 2), (2, -20)], 20) == [(7, 7, 1), (8, 8, 1)]
    assert m.map([(0, 1), (0, 1)], 20) is None and m.map([(0, 32)], 40) is None and m.map([(3, 1)], 1) is None
    assert m.map([(1, 0), (2, 0)], 0) == [] and sorted(m.free + sum(m.held, [])) == list(range(6))
    assert m.lens[1] == before[1][1]


def test_plain_attention_is_a_weighted_mean():
    r = np.random.default_rng(0)
    q, k, v = r.standard_normal((4, 8)), r.standard_normal((2, 5, 8)), r.standard_normal((2, 5, 8))
    out, off = attended(q, k, v)
    s = np.array([q[3] @ k[1, t] for t in range(5)]) / np.sqrt(8)
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(out[3], w @ v[1]) and (off > 0).all() and (off < 1e-4).all()
    assert (attended(q, k[:, :0], v[:, :0])[0] == 0).all()


def test_null_arguments_are_refused(lib):
    h = C.c_void_p()
    assert lib.shainet_paged_cache_create(None, None, 1, 1, 8, 1, 1, 0) == 1
    assert lib.shainet_paged_cache_create(C.byref(h), None, 1, 1, 8, 1, 1, 0) == 1 and not h.value
    assert b"ctx is null" in lib.shainet_hip_last_error()
    assert lib.shainet_paged_cache_destroy(None) == 0
    none6 = (None,) * 6
    assert lib.shainet_paged_cache_arrays(None, 0, *none6) == 1
    assert lib.shainet_paged_cache_map_rows(None, None, None, 1, None, None, None, 0) == 1
    assert lib.shainet_paged_cache_lengths_from_device(None) == 1
    assert lib.shainet_paged_cache_len(None, 0) == -1 and lib.shainet_paged_cache_free_pages(None) == -1
    assert lib.shainet_paged_cache_truncate(None, 0, 0) == 1 and lib.shainet_paged_cache_clear(None, -1) == 1
    assert lib.shainet_paged_cache_read(None, 0, 0, 0, 0, 1, None, None) == 1
    assert lib.shainet_attn_append_paged(None, None, 0, None, None, 1, None, 8, None, 8, None, 8, None) == 1
    assert lib.shainet_attn_attend_paged(None, None, 0, None, None, 1, None, 8, None, 8) == 1
    assert lib.shainet_attn_step_paged(None, None, 0, None, 1, None, None, None, None) == 1
    assert lib.shainet_attn_forward_paged(None, None, 0, None, None, 1, None, None, None, None, 0) == 1
    assert b"belong together" in lib.shainet_hip_last_error()


def test_lists_that_are_no_device_lists_are_refused(lib):
    import torch

    cache = hip.PagedKVCache.__new__(hip.PagedKVCache)
    cache._h, cache._handle, cache._views, cache.ctx, cache._device = None, None, {}, None, 0
    for bad in (torch.zeros(3, dtype=torch.int32), np.zeros(3, np.int32), torch.zeros(3)):
        with pytest.raises(hip.ArgumentError):
            cache.map_rows(bad)
    with pytest.raises(hip.ArgumentError, match="closed"):
        cache.table
    for bad in (torch.zeros(2, 8), np.zeros((2, 8), np.float32)):
        with pytest.raises(hip.ArgumentError):
            hip._rows(bad, 0, 2, 8)
