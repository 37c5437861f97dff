"""Attention over pages of heads whose rows no whole number of pieces fills, in sequences that hold the pool's last page."""
import numpy as np
import pytest

from test_gpu_paged import TYPES, _check_rows, _ctx, _filled, _ints, hip, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd", [(4, 4, 72), (5, 5, 80), (20, 20, 80), (6, 2, 88), (17, 1, 88), (40, 5, 88)])
def test_rows_that_end_within_a_piece(hip, torch, H, KV, hd, dtype):  # noqa: F811
    """Many short pairs, a wavefront each; a few longer ones in chunks; long ones in spans.  Every page is held by somebody."""
    rng = np.random.default_rng(hd * H)
    ctx = _ctx(hip, torch, H, KV, hd)
    for lens, P in (([1, 40, 7, 33, 32, 0] + [int(n) for n in rng.integers(1, 200, 300)], 8), ([300, 31, 450], 32), ([9000, 5, 2777], 16)):
        cache, held = _filled(hip, torch, ctx, lens, P, dtype, rng, spare=0, poison=float("nan"))
        q = rng.standard_normal((len(lens), H * hd)).astype(np.float32)
        seqs, positions = list(range(len(lens))), [n - 1 for n in lens]
        out = torch.full((len(lens), H * hd + 5), 7.0, device="cuda")
        ctx.attend_paged(cache, _ints(torch, seqs), _ints(torch, positions), torch.from_numpy(q).cuda(), out=out[:, :H * hd])
        ctx.sync()
        got = out.cpu().numpy()
        assert (got[:, H * hd:] == 7.0).all()
        _check_rows(got[:, :H * hd], q, held, seqs, positions, hd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("H,KV,hd,rows", [(16, 8, 256, 5), (6, 2, 200, 1), (8, 4, 160, 33), (3, 3, 136, 700)])
def test_rows_of_wide_heads_are_those_of_the_contiguous_cache(hip, torch, H, KV, hd, rows, norm, dtype):  # noqa: F811
    """Few and many, dense and strided: float32 pages hold the bits of a KVCache, narrow ones the same numbers rounded."""
    rng = np.random.default_rng(hd)
    f32 = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
    weights = [1 + 0.1 * f32(hd) if norm else None for _ in range(2)]
    ctx = _ctx(hip, torch, H, KV, hd, q_norm=weights[0], k_norm=weights[1])
    ctx.set_bias(f32(H * hd), f32(KV * hd), f32(KV * hd))
    q, k, v = (torch.from_numpy(f32(rows, n * hd)).cuda() for n in (H, KV, KV))
    plain = hip.KVCache(ctx, 1, rows)
    ctx.forward(plain, q, k, v, [rows])
    want = ctx.last_q_rot(rows)
    for gap in (0, 4, 3):
        cache = hip.PagedKVCache(ctx, rows // 16 + 1, 16, 1, rows // 16 + 1, dtype=dtype)
        lists = [torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(3)]
        cache.map_rows(_ints(torch, [rows]), *lists)
        wide = [torch.nn.functional.pad(x, (0, gap))[:, :x.shape[1]] for x in (q, k, v)]
        got = ctx.append_paged(cache, *lists[:2], *wide)
        cache.lengths_from_device()
        assert np.array_equal(got.cpu().numpy().view(np.uint32), want.view(np.uint32))
        for c in range(KV):
            for have, exact in zip(cache.read(0, c, 0, rows), plain.read(0, c, 0, rows)):
                assert np.array_equal(have, torch.from_numpy(exact).to(cache.k.dtype).float().numpy())
