"""Tensors over a cache's memory are of the cache's device, whichever is current: one of another would be a copy."""
import types

from shainet_amd import hip


def test_views_name_the_device_of_the_cache(monkeypatch):
    import torch

    asked = []
    monkeypatch.setattr(torch, "as_tensor", lambda array, device: asked.append((array.__cuda_array_interface__["shape"], str(device))) or torch.zeros(2, dtype=torch.int16))
    monkeypatch.setattr(hip, "lib", lambda: types.SimpleNamespace(shainet_paged_cache_arrays=lambda *a: 0))
    cache = hip.PagedKVCache.__new__(hip.PagedKVCache)
    cache._h, cache._handle, cache._views, cache._device = 1, None, {}, 3
    cache.ctx = types.SimpleNamespace(num_kv_heads=2, head_dim=8)
    cache.n_pages, cache.page_rows, cache.n_seqs, cache.seq_pages, cache.dtype = 4, 16, 5, 6, "bf16"
    for name in ("k", "v", "table", "lens", "free_pages", "n_free"):
        getattr(cache, name)
    cache.k
    cache.pages(1)
    shapes = [(4, 2, 16, 8)] * 2 + [(5, 6), (5,), (4,), (1,)] + [(4, 2, 16, 8)] * 2
    assert asked == [(shape, "cuda:3") for shape in shapes]
    cache._h = None
