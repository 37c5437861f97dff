"""Where outputs of the paged calls may lie: in the queries' place, between their rows, nowhere else among the inputs."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_paged import TYPES, _check_rows, _ctx, _filled, _ints, hip, torch  # noqa: F401

pytestmark = pytest.mark.gpu

H, KV, HD, P = 4, 2, 64, 16
W = H * HD


def _strided(torch, buffer, at, n, stride, width=W):  # noqa: F811
    return buffer.as_strided((n, width), (stride, 1), at)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride,apart", [(W, 0), (W + 8, 0), (2 * W, W), (2 * W + 4, W + 4), (3 * W, W), (W, 5 * W)])
def test_outputs_among_the_queries(hip, torch, stride, apart, dtype):  # noqa: F811
    rng = np.random.default_rng(stride + apart)
    ctx, lens = _ctx(hip, torch, H, KV, HD), [900, 3, 0, 70, 2500]
    cache, held = _filled(hip, torch, ctx, lens, P, dtype, rng)
    n = len(lens)
    rows = rng.standard_normal((n, W)).astype(np.float32)
    buffer = torch.full((20 * W + 1000,), 9.0, device="cuda")
    q, out = _strided(torch, buffer, 0, n, stride), _strided(torch, buffer, apart, n, stride)
    q.copy_(torch.from_numpy(rows))
    ctx.attend_paged(cache, _ints(torch, range(n)), _ints(torch, [x - 1 for x in lens]), q, out=out)
    ctx.sync()
    _check_rows(out.cpu().numpy(), rows, held, range(n), [x - 1 for x in lens], HD)
    if apart:
        assert np.array_equal(q.cpu().numpy(), rows)
    used = torch.zeros_like(buffer, dtype=torch.bool)
    for view in (q, out):
        used.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(True)
    assert (buffer[~used] == 9.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_at,q_stride,out_at,out_stride", [
    (0, 2 * W, W, 4 * W), (W, 4 * W, 0, 2 * W), (0, W, 5 * W, 2 * W), (0, 3 * W, W, W * 3 // 2 * 2), (10 * W, W, 0, 2 * W)])
def test_outputs_between_queries_at_another_distance(hip, torch, q_at, q_stride, out_at, out_stride, dtype):  # noqa: F811
    rng = np.random.default_rng(q_at + out_at)
    ctx, lens = _ctx(hip, torch, H, KV, HD), [700, 3, 40, 70, 1300]
    cache, held = _filled(hip, torch, ctx, lens, P, dtype, rng)
    rows = rng.standard_normal((5, W)).astype(np.float32)
    buffer = torch.full((24 * W,), 9.0, device="cuda")
    q, out = _strided(torch, buffer, q_at, 5, q_stride), _strided(torch, buffer, out_at, 5, out_stride)
    q.copy_(torch.from_numpy(rows))
    ctx.attend_paged(cache, _ints(torch, range(5)), _ints(torch, [x - 1 for x in lens]), q, out=out)
    ctx.sync()
    _check_rows(out.cpu().numpy(), rows, held, range(5), [x - 1 for x in lens], HD)
    assert np.array_equal(q.cpu().numpy(), rows)


@pytest.mark.parametrize("q_at,q_stride,out_at,out_stride", [
    (0, 2 * W, W, 3 * W), (0, 3 * W, 2 * W - 4, 4 * W), (4 * W, 2 * W, 0, W * 9 // 4), (0, W, 0, W + 4), (0, 2 * W, 0, W), (0, W, 4, W), (0, W, W, W), (4, W, 0, W), (0, 2 * W, W - 4, 2 * W), (0, 2 * W, W + 4, 2 * W),
    (0, W, 2 * W + 4, W), (2 * W, W, 0, 2 * W)])
def test_outputs_in_the_way_of_queries(hip, torch, q_at, q_stride, out_at, out_stride):  # noqa: F811
    ctx = _ctx(hip, torch, H, KV, HD)
    cache = hip.PagedKVCache(ctx, 4, P, 3, 2, dtype="f32")
    buffer = torch.full((24 * W,), 9.0, device="cuda")
    q, out = _strided(torch, buffer, q_at, 3, q_stride), _strided(torch, buffer, out_at, 3, out_stride)
    three = _ints(torch, [0, 1, 2])
    with pytest.raises(hip.ArgumentError, match="apart"):
        ctx.attend_paged(cache, three, three, q, out=out)
    one = _ints(torch, [0])
    if 0 < abs(q_at - out_at) < W:
        with pytest.raises(hip.ArgumentError, match="apart"):
            ctx.attend_paged(cache, one, one, q[:1], out=out[:1])
    else:
        ctx.attend_paged(cache, one, one, q[:1], out=out[:1])
    ctx.sync()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,norm", [(5, False), (5, True), (900, False), (900, True)])
def test_rotated_queries_in_their_place(hip, torch, rows, norm, dtype):  # noqa: F811
    """As few rows, as many, with and without QK-norm, are placed: the same bits as with a place of their own."""
    rng = np.random.default_rng(rows)
    weights = [(1 + 0.1 * rng.standard_normal(HD)).astype(np.float32) if norm else None for _ in range(2)]
    ctx = _ctx(hip, torch, H, KV, HD, q_norm=weights[0], k_norm=weights[1])
    cache = hip.PagedKVCache(ctx, 60, P, 1, 60, dtype=dtype)
    q, k, v = (torch.from_numpy(rng.standard_normal((rows, w * HD)).astype(np.float32)).cuda() for w in (H, KV, KV))
    lists = _ints(torch, range(rows)), _ints(torch, range(rows))
    want = ctx.append_paged(cache, *lists, q, k, v)
    pages = [t.clone() for t in cache.pages(0)]
    got = ctx.append_paged(cache, *lists, q, k, v, q_rot=q)
    ctx.sync()
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(pages, cache.pages(0)))


def test_rotated_queries_in_the_way(hip, torch):  # noqa: F811
    ctx = _ctx(hip, torch, H, KV, HD)
    cache = hip.PagedKVCache(ctx, 4, P, 1, 4)
    buffer = torch.zeros(40 * W, device="cuda")
    lists = _ints(torch, range(3)), _ints(torch, range(3))
    half = KV * HD
    fused = W + 2 * half  # rows of q, k and v side by side
    q, k, v = (_strided(torch, buffer, at, 3, fused, width) for at, width in ((0, W), (W, half), (W + half, half)))
    for at in (0, W, 2 * fused, 3 * fused - half - W, 3 * fused - 4):
        with pytest.raises(hip.ArgumentError, match="apart"):
            ctx.append_paged(cache, *lists, q, k, v, q_rot=_strided(torch, buffer, at, 3, W))
    ctx.append_paged(cache, *lists, q, k, v, q_rot=_strided(torch, buffer, 3 * fused, 3, W))
    ctx.sync()
