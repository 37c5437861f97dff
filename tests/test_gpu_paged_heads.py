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
