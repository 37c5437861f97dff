"""A KV cache in pages on the GPU: maps of slots, new rows into them, attention over them, and the three together, against
plain Python in 64 bits and against the contiguous cache."""
import numpy as np
import pytest

from paged_model import Pages, attended, pages_of, turned

pytestmark = pytest.mark.gpu

TYPES = ("f32", "bf16", "f16")


@pytest.fixture(scope="module")
def hip():
    import shainet_amd as sa

    assert sa.HIP.fully_available(), "no gfx950 device or libshainet_hip_kernels.so missing"
    return sa


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _ints(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ctx(hip, torch, H, KV, hd, **more):
    ctx = hip.AttnContext(H, KV, hd, rope_theta=1e6, **more)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return ctx


# ---- maps ---------------------------------------------------------------------------------------

def _same_state(cache, model, n_free):
    table, lens, free = cache.table.cpu().numpy(), cache.lens.cpu().numpy(), cache.free_pages.cpu().numpy()
    assert cache.n_free.item() == n_free == len(model.free)
    assert lens.tolist() == model.lens
    assert free[:n_free].tolist() == model.free
    for s, held in enumerate(model.held):
        assert table[s, :len(held)].tolist() == held, s


# pages, rows a page, sequences, table width, lists: the last three are moved by a launch of many workgroups
MAPS = [(40, 8, 5, 12, 64), (64, 16, 1, 64, 300), (300, 8, 130, 9, 700), (2000, 32, 1100, 4, 4000), (5000, 8, 4096, 2, 5000),
        (20000, 8, 300, 100, 300), (900, 1024, 20, 60, 60000), (17000, 16, 4096, 17, 50000)]


@pytest.mark.parametrize("n_pages,P,n_seqs,seq_pages,max_rows", MAPS)
def test_maps_follow_the_plain_ones(hip, torch, n_pages, P, n_seqs, seq_pages, max_rows):
    rng = np.random.default_rng(n_pages + P)
    cache = hip.PagedKVCache(_ctx(hip, torch, 1, 1, 8), n_pages, P, n_seqs, seq_pages)
    model = Pages(n_pages, P, n_seqs, seq_pages)
    lists = [torch.empty(max_rows, dtype=torch.int32, device="cuda") for _ in range(3)]
    for turn in range(12):
        n = int(rng.integers(1, n_seqs + 1))
        seqs = rng.permutation(n_seqs)[:n]
        room = min(P * seq_pages, max(1, 2 * n_pages * P // n_seqs), max(1, 2 * max_rows // n))
        entries = []
        for s in seqs.tolist():
            kind = rng.integers(0, 5)
            d = (1, 0, -model.lens[s], int(rng.integers(0, room + 1)), -int(rng.integers(0, model.lens[s] + 1)))[kind]
            entries.append((s, min(d, P * seq_pages - model.lens[s])))
        if turn == 11:  # from nothing: tables made of the lengths alone
            cache.clear()
            model = Pages(n_pages, P, n_seqs, seq_pages)
            entries = [(s, d) for s, d in entries if d >= 0] or [(0, 1)]
        for t in lists:
            t.fill_(-7)
        rows = model.map(entries, max_rows)
        cache.map_rows(_ints(torch, [d for _, d in entries]), *lists, seq_ids=_ints(torch, [s for s, _ in entries]))
        want = np.full((max_rows, 3), -1)
        if rows:
            want[:len(rows)] = rows
        got = np.stack([t.cpu().numpy() for t in lists], 1)
        assert np.array_equal(got, want), (turn, rows is None)
        _same_state(cache, model, len(model.free))
        if rows is None:
            with pytest.raises(hip.HipError, match="map of new rows"):
                cache.lengths_from_device()
        else:
            cache.lengths_from_device()
        assert [cache.len(s) for s in range(n_seqs)] == model.lens and cache.free_page_count() == len(model.free)


@pytest.mark.parametrize("big", [False, True])
def test_a_map_and_its_inverse_leave_everything(hip, torch, big):
    n_pages, P, n = (30000, 8, 700) if big else (3000, 8, 70)
    cache = hip.PagedKVCache(_ctx(hip, torch, 1, 1, 8), n_pages, P, n, 60)
    rng = np.random.default_rng(3)
    first = _ints(torch, rng.integers(0, 200, n))
    lists = [torch.empty(n * 400, dtype=torch.int32, device="cuda") for _ in range(3)]
    cache.map_rows(first, *lists)
    before = [t.clone() for t in (cache.lens, cache.n_free, cache.free_pages)]
    held = cache.table.clone()
    change = torch.where(_ints(torch, rng.integers(0, 2, n)) > 0, -first, _ints(torch, rng.integers(0, 200, n)))
    order = _ints(torch, rng.permutation(n))
    d = change[order.long()].contiguous()
    cache.map_rows(d, *lists, seq_ids=order)
    assert not torch.equal(cache.lens, before[0])
    cache.map_rows(-d, *lists, seq_ids=order)
    cache.lengths_from_device()
    top = before[1].item()
    assert torch.equal(cache.lens, before[0]) and torch.equal(cache.n_free, before[1])
    assert torch.equal(cache.free_pages[:top], before[2][:top])
    for s in range(n):
        p = pages_of(first[s].item(), P)
        assert torch.equal(cache.table[s, :p], held[s, :p])


def _refused(hip, torch, cache, entries, error, lists):
    state = [t.clone() for t in (cache.table, cache.lens, cache.free_pages, cache.n_free)]
    cache.map_rows(_ints(torch, [d for _, d in entries]), *lists, seq_ids=_ints(torch, [s for s, _ in entries]))
    for was, now in zip(state, (cache.table, cache.lens, cache.free_pages, cache.n_free)):
        assert torch.equal(was, now)
    for t in lists:
        assert (t == -1).all()
    with pytest.raises(error):
        cache.ctx.sync()
    cache.ctx.sync()  # said once


@pytest.mark.parametrize("max_rows", [64, 9000])
def test_maps_that_cannot_be_made_change_nothing(hip, torch, max_rows):
    cache = hip.PagedKVCache(_ctx(hip, torch, 1, 1, 8), 10, 8, 4, 6)
    lists = [torch.empty(max_rows, dtype=torch.int32, device="cuda") for _ in range(3)]
    cache.map_rows(_ints(torch, [30, 9]), *lists)
    for entries, error in (([(2, 40)], hip.HipError),             # 4 pages are left
                           ([(1, 45)], hip.HipError),             # more than a table row holds
                           ([(0, 1), (4, 1)], hip.ArgumentError),  # no such sequence
                           ([(-1, 1)], hip.ArgumentError),
                           ([(3, 1), (3, 1)], hip.ArgumentError),  # twice
                           ([(0, -31)], hip.ArgumentError),        # below 0
                           ([(0, 2 ** 31 - 1)], hip.HipError),
                           ([(0, -2 ** 31)], hip.ArgumentError)):
        _refused(hip, torch, cache, entries, error, lists)
    few = [t[:3] for t in lists]
    _refused(hip, torch, cache, [(2, 4)], hip.HipError, few)
    cache.map_rows(_ints(torch, [-30, 40]), *lists, seq_ids=_ints(torch, [0, 2]))  # what one gives back the other takes
    cache.lengths_from_device()
    assert [cache.len(s) for s in range(4)] == [0, 9, 40, 0] and cache.free_page_count() == 3


# ---- new rows into their slots --------------------------------------------------------------------

ROWS = [  # H, KV, hd, rows, page rows, QK-norm, biases
    (4, 2, 8, 1, 8, False, False),
    (8, 2, 64, 5, 16, False, True),
    (32, 8, 128, 16, 16, True, False),
    (5, 5, 80, 33, 8, True, True),
    (6, 2, 200, 9, 32, True, True),     # heads wider than a wavefront's pairs
    (4, 4, 256, 7, 64, False, False),
    (32, 8, 64, 400, 16, False, False),  # enough for four pairs a lane
    (32, 8, 64, 400, 16, False, True),
    (32, 8, 128, 300, 128, True, True),  # enough for rows through LDS
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd,rows,P,norm,bias", ROWS)
def test_new_rows_land_in_their_slots(hip, torch, H, KV, hd, rows, P, norm, bias, dtype):
    rng = np.random.default_rng(H * hd + rows)
    f32 = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
    qn, kn = (1 + 0.1 * f32(hd), 1 + 0.1 * f32(hd)) if norm else (None, None)
    bq, bk, bv = (f32(H * hd), f32(KV * hd), f32(KV * hd)) if bias else (None, None, None)
    ctx = _ctx(hip, torch, H, KV, hd, q_norm=qn, k_norm=kn)
    ctx.set_bias(bq, bk, bv)
    n_pages, far = pages_of(rows, P) + 3, 2000
    cache = hip.PagedKVCache(ctx, n_pages, P, 1, pages_of(far, P), dtype=dtype)
    for pool in (cache.k, cache.v):
        pool.copy_(torch.from_numpy(f32(*pool.shape)))
    before = [cache.k.clone(), cache.v.clone()]
    slots = rng.permutation(n_pages * P)[:rows]
    positions = rng.integers(0, far, rows)
    skipped = sorted(rng.permutation(rows)[:rows // 4].tolist())
    for i, r in enumerate(skipped):
        if i % 2:
            slots[r] = (-1, n_pages * P, -2 ** 31, 2 ** 31 - 1)[i // 2 % 4]
        else:
            positions[r] = (-1, 2 ** 31 - 1, -2 ** 31)[i // 2 % 3]
    q, k, v = f32(rows, H * hd), f32(rows, KV * hd), f32(rows, KV * hd)
    # rows 7 numbers apart, then dense ones
    for gap in (7, 0):
        wide = [torch.from_numpy(np.pad(x, ((0, 0), (0, gap)))).cuda()[:, :x.shape[1]] for x in (q, k, v)]
        q_rot = torch.full((rows, H * hd), 9.0, device="cuda")
        for pool, was in zip((cache.k, cache.v), before):
            pool.copy_(was)
        ctx.append_paged(cache, _ints(torch, slots), _ints(torch, positions), *wide, q_rot=q_rot)
        ctx.sync()
        kept = [r for r in range(rows) if r not in skipped]
        freq = ctx.inv_freq()
        want = [turned(x[kept], hd, positions[kept], freq, w, b) for x, w, b in ((q, qn, bq), (k, kn, bk))]
        want.append((v[kept].astype(np.float64) + (0 if bv is None else bv)))
        # u = 2^-24: bias 1 u; the mean of squares (hd + 2) u, halved by the root, and 3 u of root, quotient and rounding; three products and
        # the rotation's sum; cos and sin 2 u each; against the largest pair
        size = lambda x: np.abs(x.reshape(len(x), -1, hd)).max(-1, keepdims=True).repeat(hd, -1).reshape(x.shape)  # noqa: E731
        off = lambda x: 2.0 ** -24 * (hd / 2 + 16 if norm else 10) * 2 * size(x) + 1e-12  # noqa: E731
        got = q_rot.cpu().numpy()
        assert (np.abs(got[kept] - want[0]) <= off(want[0])).all()
        assert (got[skipped] == 9.0).all()
        half = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
        for pool, was, exact in ((cache.k, before[0], want[1]), (cache.v, before[1], want[2])):
            flat = pool.transpose(1, 2).reshape(-1, KV * hd).float().cpu().numpy()
            rest = was.transpose(1, 2).reshape(-1, KV * hd).float().cpu().numpy()
            at = slots[kept]
            assert (np.abs(flat[at] - exact) <= off(exact) + half * (np.abs(exact) + off(exact)) + (2.0 ** -25 if dtype == "f16" else 0)).all()
            others = np.setdiff1d(np.arange(n_pages * P), at)
            assert np.array_equal(flat[others], rest[others])


@pytest.mark.parametrize("H,KV,hd,norm,bias", [(32, 8, 128, True, False), (8, 2, 64, False, True), (5, 5, 80, True, True)])
@pytest.mark.parametrize("rows", [3, 400])
def test_rows_are_those_of_the_contiguous_cache(hip, torch, H, KV, hd, norm, bias, rows):
    """Float32 pages hold the bits that a KVCache holds, narrow ones the same numbers rounded to the nearest."""
    rng = np.random.default_rng(5)
    f32 = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
    qn, kn = (1 + 0.1 * f32(hd), 1 + 0.1 * f32(hd)) if norm else (None, None)
    ctx = _ctx(hip, torch, H, KV, hd, q_norm=qn, k_norm=kn)
    if bias:
        ctx.set_bias(f32(H * hd), f32(KV * hd), f32(KV * hd))
    q, k, v = (torch.from_numpy(f32(rows, n * hd)).cuda() for n in (H, KV, KV))
    plain = hip.KVCache(ctx, 1, rows)
    ctx.forward(plain, q, k, v, [rows])
    q_rot = ctx.last_q_rot(rows)
    for dtype in TYPES:
        cache = hip.PagedKVCache(ctx, pages_of(rows, 16), 16, 1, pages_of(rows, 16), dtype=dtype)
        lists = [torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(3)]
        cache.map_rows(_ints(torch, [rows]), *lists)
        got = ctx.append_paged(cache, *lists[:2], q, k, v)
        cache.lengths_from_device()
        assert np.array_equal(got.cpu().numpy().view(np.uint32), q_rot.view(np.uint32))
        for c in range(KV):
            for have, want in zip(cache.read(0, c, 0, rows), plain.read(0, c, 0, rows)):
                want = torch.from_numpy(want).to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype])
                assert np.array_equal(have, want.float().numpy())


# ---- attention ------------------------------------------------------------------------------------

def _filled(hip, torch, ctx, lens, P, dtype, rng, spare=3, poison=None, spread=1.0):
    """A cache of sequences of these lengths in scattered pages; the rows of each as [KV, n, hd] of the pages' numbers.
    poison: what all other rows of the pool hold."""
    KV, hd = ctx.num_kv_heads, ctx.head_dim
    counts = [pages_of(n, P) for n in lens]
    n_pages = sum(counts) + spare
    cache = hip.PagedKVCache(ctx, n_pages, P, len(lens), max(1, max(counts)), dtype=dtype)
    order = rng.permutation(n_pages)
    table = rng.integers(-5, n_pages + 5, (len(lens), cache.seq_pages))  # behind the last page: anything
    pools = [np.full((n_pages, KV, P, hd), 0.0 if poison is None else poison, np.float32) for _ in range(2)]
    held, at = [], 0
    for s, n in enumerate(lens):
        pages = order[at:at + counts[s]]
        at += counts[s]
        table[s, :counts[s]] = pages
        rows = [(spread * rng.standard_normal((KV, n, hd))).astype(np.float32) for _ in range(2)]
        rows = [torch.from_numpy(x).to(cache.k.dtype).float().numpy() for x in rows]
        for pool, x in zip(pools, rows):
            for i, page in enumerate(pages):
                part = x[:, i * P:(i + 1) * P]
                pool[page, :, :part.shape[1]] = part
        held.append(rows)
    cache.k.copy_(torch.from_numpy(pools[0]))
    cache.v.copy_(torch.from_numpy(pools[1]))
    cache.table.copy_(torch.from_numpy(table.astype(np.int32)))
    return cache, held


def _check_rows(got, q, held, row_seqs, positions, hd):
    for r, (s, p) in enumerate(zip(row_seqs, positions)):
        k, v = (x[:, :p + 1] for x in held[s]) if p >= 0 else (x[:, :0] for x in held[s])
        want, off = attended(q[r].reshape(-1, hd), k, v)
        off = np.maximum(off, 2.0 ** -23 * np.abs(want))
        worst = (np.abs(got[r].reshape(-1, hd) - want) / np.maximum(off, 1e-30)).max()
        assert worst <= 1, (r, s, p, worst)


HEADS = [(1, 1, 8), (4, 4, 64), (8, 2, 64), (32, 8, 128), (7, 1, 96), (14, 2, 80), (16, 1, 128), (17, 1, 64), (40, 2, 72), (48, 1, 128),
         (6, 2, 256), (4, 1, 160), (3, 3, 24)]
EDGES = [0, 1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257, 700]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd", HEADS)
def test_attention_of_every_head_geometry(hip, torch, H, KV, hd, dtype):
    rng = np.random.default_rng(H * 1000 + hd)
    ctx = _ctx(hip, torch, H, KV, hd)
    P = int(rng.choice([8, 16, 32]))
    cache, held = _filled(hip, torch, ctx, EDGES, P, dtype, rng, poison=float("nan"))
    q = rng.standard_normal((len(EDGES), H * hd)).astype(np.float32)
    seqs, positions = list(range(len(EDGES))), [n - 1 for n in EDGES]
    got = ctx.attend_paged(cache, _ints(torch, seqs), _ints(torch, positions), torch.from_numpy(q).cuda())
    ctx.sync()
    _check_rows(got.cpu().numpy(), q, held, seqs, positions, hd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P", [8, 16, 32, 64, 128, 256, 512, 1024])
def test_attention_over_every_page_size(hip, torch, P, dtype):
    H, KV, hd = 8, 2, 128
    rng = np.random.default_rng(P)
    ctx = _ctx(hip, torch, H, KV, hd)
    lens = [P - 1, P, P + 1, 2 * P + 5, 3, 1500]
    cache, held = _filled(hip, torch, ctx, lens, P, dtype, rng, poison=float("inf"))
    q = rng.standard_normal((len(lens), H * hd)).astype(np.float32)
    seqs, positions = list(range(len(lens))), [n - 1 for n in lens]
    got = ctx.attend_paged(cache, _ints(torch, seqs), _ints(torch, positions), torch.from_numpy(q).cuda())
    ctx.sync()
    _check_rows(got.cpu().numpy(), q, held, seqs, positions, hd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd,lens,P", [
    (32, 8, 64, [20000], 16),               # one sequence over many workgroups
    (16, 2, 128, [30011, 5, 9000], 64),
    (4, 1, 256, [12345], 8),
    (32, 4, 128, [3000, 1, 0, 2999] + [40] * 60, 32),
    (8, 8, 64, [17] * 300, 16),             # many short ones
    (2, 1, 16, [1] * 1025 + [50], 8),       # more rows than a workgroup has threads
])
def test_long_and_many_sequences(hip, torch, H, KV, hd, lens, P, dtype):
    rng = np.random.default_rng(len(lens))
    ctx = _ctx(hip, torch, H, KV, hd)
    cache, held = _filled(hip, torch, ctx, lens, P, dtype, rng, poison=float("nan"))
    q = rng.standard_normal((len(lens), H * hd)).astype(np.float32)
    seqs, positions = list(range(len(lens))), [n - 1 for n in lens]
    args = _ints(torch, seqs), _ints(torch, positions), torch.from_numpy(q).cuda()
    got = ctx.attend_paged(cache, *args)
    again = ctx.attend_paged(cache, *args)
    ctx.sync()
    _check_rows(got.cpu().numpy(), q, held, seqs, positions, hd)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_in_any_order_and_rows_left_alone(hip, torch, dtype):
    H, KV, hd, P = 8, 4, 64, 16
    rng = np.random.default_rng(8)
    ctx = _ctx(hip, torch, H, KV, hd)
    lens = [300, 40, 7, 129]
    cache, held = _filled(hip, torch, ctx, lens, P, dtype, rng, poison=float("nan"))
    seqs = [3, 0, 0, 0, 2, -1, 1, 4, 0, 3, -2 ** 31, 2 ** 31 - 1, 1]
    positions = [128, 299, 10, 0, -1, 5, 39, 3, 150, 60, 4, 4, -100]
    n = len(seqs)
    q = rng.standard_normal((n, H * hd + 6)).astype(np.float32)
    out = torch.full((n, H * hd + 2), 5.0, device="cuda")
    ctx.attend_paged(cache, _ints(torch, seqs), _ints(torch, positions), torch.from_numpy(q).cuda()[:, :H * hd], out=out[:, :H * hd])
    ctx.sync()
    got = out.cpu().numpy()
    assert (got[:, H * hd:] == 5.0).all()
    kept = [r for r in range(n) if 0 <= seqs[r] < 4]
    assert (got[[r for r in range(n) if r not in kept]] == 5.0).all()
    _check_rows(got[kept][:, :H * hd], q[kept][:, :H * hd], held, [seqs[r] for r in kept], [positions[r] for r in kept], hd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,P", [(64, 8), (128, 16), (128, 64), (256, 32)])
def test_keys_of_pages_outside_the_pool_take_no_part(hip, torch, hd, P, dtype):
    H, KV = 6, 2
    rng = np.random.default_rng(hd + P)
    ctx = _ctx(hip, torch, H, KV, hd)
    lens = [400, 5 * P, P, 3]
    cache, held = _filled(hip, torch, ctx, lens, P, dtype, rng, poison=float("nan"))
    table = cache.table.cpu().numpy()
    gone = [(0, 1), (0, pages_of(400, P) - 1), (1, 0), (1, 2), (1, 3), (2, 0)]
    for (s, i), bad in zip(gone, (-1, cache.n_pages, 2 ** 31 - 1, -2 ** 31, cache.n_pages + 1, -1)):
        table[s, i] = bad
    cache.table.copy_(torch.from_numpy(table))
    for s, rows in enumerate(held):
        keep = [t for t in range(lens[s]) if (s, t // P) not in gone]
        held[s] = [x[:, keep] for x in rows]
    q = rng.standard_normal((4, H * hd)).astype(np.float32)
    got = ctx.attend_paged(cache, _ints(torch, range(4)), _ints(torch, [n - 1 for n in lens]), torch.from_numpy(q).cuda())
    ctx.sync()
    _check_rows(got.cpu().numpy(), q, held, range(4), [x[0].shape[1] - 1 for x in held], hd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e-30, 1e-4, 30.0, 1e4])
def test_queries_small_and_large(hip, torch, size, dtype):
    """From weights that are all alike to one key that counts alone; lengths beyond the table's width are cut to it."""
    H, KV, hd, P = 8, 2, 128, 16
    rng = np.random.default_rng(21)
    ctx = _ctx(hip, torch, H, KV, hd)
    lens = [512, 512, 90]
    cache, held = _filled(hip, torch, ctx, lens, P, dtype, rng)
    q = (size * rng.standard_normal((3, H * hd))).astype(np.float32)
    q[0, ::3] *= 1e-6  # parts of very different sizes
    got = ctx.attend_paged(cache, _ints(torch, range(3)), _ints(torch, [2 ** 31 - 1, 511, 89]), torch.from_numpy(q).cuda())
    ctx.sync()
    _check_rows(got.cpu().numpy(), q, held, range(3), [511, 511, 89], hd)


# ---- together -------------------------------------------------------------------------------------

def _tolerance(dtype):
    # keys and values rounded to the pages' type: a score is off by a half step of |q| |k| / sqrt(hd), a value by one of itself;
    # inputs of size 1 and QK-norm: scores up to about 4 sqrt(hd) / sqrt(hd) * a few
    return {"f32": 2e-5, "bf16": 0.1, "f16": 0.0125}[dtype]


@pytest.mark.parametrize("n_pages,short", [(40, False), (24, True)])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_server_of_requests_that_come_and_go(hip, torch, dtype, n_pages, short):
    """Prompts, steps and ends of requests over a pool that holds few of them; every output against a contiguous cache of that request alone."""
    H, KV, hd, P = 8, 2, 64, 16
    rng = np.random.default_rng(77)
    qn, kn = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32), (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    ctx = _ctx(hip, torch, H, KV, hd, q_norm=qn, k_norm=kn)
    slots = 4
    cache = hip.PagedKVCache(ctx, n_pages, P, slots, 20, dtype=dtype)
    alone = [hip.KVCache(ctx, 1, 320) for _ in range(slots)]
    new = lambda n: [torch.from_numpy(rng.standard_normal((n, w * hd)).astype(np.float32)).cuda() for w in (H, KV, KV)]  # noqa: E731
    live, refused = {}, 0
    worst = 0.0
    for turn in range(60):
        entries = []
        for s in rng.permutation(slots).tolist():
            if s not in live:
                entries.append((s, int(rng.choice([1, 2, 5, 17, 40, 130, 200]))))
            elif rng.random() < 0.1 or live[s] > 290:
                cache.clear(s)
                alone[s].clear()
                del live[s]
            else:
                entries.append((s, int(rng.choice([1, 1, 1, 3, 6]))))
        if not entries:
            continue
        if turn % 3 == 0:  # a step of one row each, planned on the device
            entries = [(s, 1) for s, _ in entries]
        q, k, v = new(sum(d for _, d in entries))
        try:
            if turn % 3 == 0:
                got = ctx.step_paged(cache, q, k, v, torch.full_like(q, 3.0), seq_ids=_ints(torch, [s for s, _ in entries]))
                cache.lengths_from_device()
            else:
                got = ctx.forward_paged(cache, q, k, v, [d for _, d in entries], seq_ids=[s for s, _ in entries])
        except hip.HipError as e:
            assert "pages" in str(e) and sum(pages_of(live.get(s, 0) + d, P) - pages_of(live.get(s, 0), P) for s, d in entries) > cache.free_page_count()
            refused += 1
            continue
        at = 0
        for s, d in entries:
            want = ctx.forward(alone[s], *(x[at:at + d].contiguous() for x in (q, k, v)), [d])
            ctx.sync()
            worst = max(worst, (got[at:at + d] - want).abs().max().item())
            live[s] = live.get(s, 0) + d
            assert cache.len(s) == live[s] == alone[s].len(0)
            at += d
        assert cache.free_page_count() == n_pages - sum(pages_of(n, P) for n in live.values())
    assert worst <= _tolerance(dtype) and (refused > 0) == short
    for s, n in live.items():
        kp, vp = cache.read(s, 1, 0, n)
        kc, vc = alone[s].read(0, 1, 0, n)
        if dtype == "f32":
            assert np.array_equal(kp, kc) and np.array_equal(vp, vc)
        else:
            assert np.abs(kp - kc).max() <= 2.0 ** -8 * np.abs(kc).max() and np.abs(vp - vc).max() <= 2.0 ** -8 * np.abs(vc).max()


@pytest.mark.parametrize("dtype", TYPES)
def test_recorded_steps_of_two_layers(hip, torch, dtype):
    """A step of two layers recorded once and replayed, with eager work between the replays; the last replays find no page."""
    H, KV, hd, P, n = 8, 2, 128, 8, 5
    rng = np.random.default_rng(1)
    stream = torch.cuda.Stream()
    sides = []
    for _ in range(2):
        ctxs = [hip.AttnContext(H, KV, hd, rope_theta=1e6) for _ in range(2)]  # (tables of 1024 positions: they reach)
        for c in ctxs:
            c.set_stream(stream.cuda_stream)
        sides.append((ctxs, hip.PagedKVCache(ctxs[0], 23, P, 7, 6, dtype=dtype, layers=2)))
    ids = _ints(torch, [6, 0, 3, 2, 5])
    x = [[torch.empty((n, w * hd), device="cuda") for w in (H, KV, KV)] for _ in range(2)]
    outs = [[torch.zeros((n, H * hd), device="cuda") for _ in range(2)] for _ in range(2)]
    fresh = lambda: [t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32))) for layer in x for t in layer]  # noqa: E731

    def step(side):
        ctxs, cache = sides[side]
        for layer in range(2):
            ctxs[layer].step_paged(cache, *x[layer], outs[side][layer], seq_ids=ids, layer=layer)

    for side in range(2):
        for s, d in ((6, 17), (3, 7), (2, 8)):
            gen = np.random.default_rng(s)
            rows = [gen.standard_normal((d, w * hd)).astype(np.float32) for w in (H, KV, KV)]
            for layer in range(2):
                sides[side][0][layer].forward_paged(sides[side][1], *rows, [d], seq_ids=[s], layer=layer)
    fresh()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(1)
    lens = {6: 17, 0: 0, 3: 7, 2: 8, 5: 0}
    ended = 0
    for turn in range(29):  # 25 steps fill 23 pages: 6 + 4 + 4 + 4 + 5
        fresh()
        torch.cuda.synchronize()
        step(0)
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        errors = 0
        for ctxs, cache in sides:
            try:
                cache.lengths_from_device()
            except hip.HipError as e:
                assert "free pages" in str(e)
                errors += 1
                cache.lengths_from_device()
        assert errors in (0, 2)
        ended += errors == 2
        for s in lens:
            lens[s] += 0 if errors else 1
            assert sides[0][1].len(s) == sides[1][1].len(s) == lens[s]
        for layer in range(2):
            assert torch.equal(outs[0][layer], outs[1][layer]), (turn, layer)
            for c in range(KV):
                for s in lens:
                    a, b = (cache.read(s, c, 0, lens[s], layer=layer) for _, cache in sides)
                    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    assert ended == 4


def test_the_host_mode_and_several_layers(hip, torch):
    H, KV, hd, P = 4, 2, 64, 8
    rng = np.random.default_rng(4)
    ctx, other = _ctx(hip, torch, H, KV, hd), _ctx(hip, torch, H, KV, hd, q_norm=np.ones(hd, np.float32), k_norm=np.ones(hd, np.float32))
    cache = hip.PagedKVCache(ctx, 30, P, 3, 10, dtype="f32", layers=2)
    plain = [hip.KVCache(c, 3, 80) for c in (ctx, other)]
    for turn, (ids, new) in enumerate([([0, 2], [20, 1]), ([2, 0, 1], [1, 4, 30]), ([1], [1]), ([0, 1, 2], [5, 1, 12])]):
        for layer, c in enumerate((ctx, other)):
            rows = [rng.standard_normal((sum(new), w * hd)).astype(np.float32) for w in (H, KV, KV)]
            got = c.forward_paged(cache, *rows, new, seq_ids=ids, layer=layer)
            want = c.forward(plain[layer], *rows, new, seq_ids=ids)
            assert np.abs(got - want).max() <= 2e-5, (turn, layer)
    for layer in range(2):
        for s in range(3):
            assert cache.len(s) == plain[layer].len(s)
            for c in range(KV):
                for a, b in zip(cache.read(s, c, 0, cache.len(s), layer=layer), plain[layer].read(s, c, 0, cache.len(s))):
                    assert np.array_equal(a, b)
    with pytest.raises(hip.ArgumentError, match="layer 0"):  # other rows than layer 0 mapped
        other.forward_paged(cache, *rows, [5, 12, 1], seq_ids=ids, layer=1)


def test_calls_that_are_refused(hip, torch):
    H, KV, hd = 4, 2, 64
    ctx = _ctx(hip, torch, H, KV, hd)
    for bad in ((4, 7, 2, 2), (4, 12, 2, 2), (4, 2048, 2, 2), (0, 8, 2, 2), (4, 8, 0, 2), (4, 8, 4097, 2), (4, 8, 2, 0),
                (2 ** 30, 8, 2, 2), (4, 1024, 1, 2 ** 21), (4, 8, 4096, 2 ** 20)):
        with pytest.raises(hip.ArgumentError):
            hip.PagedKVCache(ctx, *bad)
    with pytest.raises(hip.ArgumentError):
        hip.PagedKVCache(ctx, 4, 8, 2, 2, dtype="f64")
    with pytest.raises(hip.ArgumentError):
        hip.PagedKVCache(_ctx(hip, torch, 2, 2, 60), 4, 8, 2, 2)
    cache = hip.PagedKVCache(ctx, 4, 8, 2, 3)
    rows = lambda n: [torch.zeros((n, w * hd), device="cuda") for w in (H, KV, KV)]  # noqa: E731
    one = _ints(torch, [0])
    with pytest.raises(hip.ArgumentError, match="belong together"):
        _ctx(hip, torch, 4, 4, 64).attend_paged(cache, one, one, rows(1)[0])
    with pytest.raises(hip.ArgumentError, match="more query heads"):
        _ctx(hip, torch, 8, 2, 64).attend_paged(cache, one, one, torch.zeros((1, 512), device="cuda"))
    with pytest.raises(hip.ArgumentError, match="one stream"):
        hip.AttnContext(H, KV, hd).attend_paged(cache, one, one, rows(1)[0])
    with pytest.raises(hip.ArgumentError, match="layer"):
        ctx.attend_paged(cache, one, one, rows(1)[0], layer=1)
    with pytest.raises(hip.ArgumentError, match="rows must be"):
        many = torch.zeros(4097, dtype=torch.int32, device="cuda")
        ctx.attend_paged(cache, many, many, torch.zeros((4097, H * hd), device="cuda"))
    with pytest.raises(hip.ArgumentError):
        ctx.attend_paged(cache, one.long(), one, rows(1)[0])
    with pytest.raises(hip.ArgumentError):
        ctx.attend_paged(cache, one, one, rows(1)[0].double())
    with pytest.raises(hip.ArgumentError):
        ctx.append_paged(cache, one, one, *rows(2))
    with pytest.raises(hip.ArgumentError):
        cache.map_rows(_ints(torch, [1, 1, 1]))
    with pytest.raises(hip.ArgumentError):
        cache.map_rows(one, slots=one)
    with pytest.raises(hip.ArgumentError, match="new_tokens"):
        ctx.forward_paged(cache, *rows(1), [1, 0])
    with pytest.raises(hip.ArgumentError, match="twice"):
        ctx.forward_paged(cache, *rows(2), [1, 1], seq_ids=[1, 1])
    with pytest.raises(hip.ArgumentError, match="out of range"):
        ctx.forward_paged(cache, *rows(1), [1], seq_ids=[2])
    with pytest.raises(hip.HipError, match="exceed"):
        ctx.forward_paged(cache, *rows(25), [25])
    with pytest.raises(hip.HipError, match="free"):
        ctx.forward_paged(cache, *rows(33), [17, 16])
    with pytest.raises(hip.ArgumentError, match="layer 0"):
        hip.PagedKVCache(ctx, 4, 8, 2, 3, layers=2) and ctx.forward_paged(hip.PagedKVCache(ctx, 4, 8, 2, 3, layers=2), *rows(1), [1], layer=1)
    assert cache.len(0) == 0 and cache.free_page_count() == 4
    ctx.forward_paged(cache, *rows(20), [20])
    assert cache.free_page_count() == 1
    cache.map_rows(_ints(torch, [1]), *(torch.empty(1, dtype=torch.int32, device="cuda") for _ in range(3)), seq_ids=_ints(torch, [1]))
    assert cache.len(0) == -1 and cache.free_page_count() == -1
    for call in (lambda: ctx.forward_paged(cache, *rows(1), [1]), lambda: cache.truncate(0, 3), lambda: cache.read(0, 0, 0, 1)):
        with pytest.raises(hip.ArgumentError, match="lengths_from_device"):
            call()
    cache.lengths_from_device()
    assert (cache.len(0), cache.len(1), cache.free_page_count()) == (20, 1, 0)
    with pytest.raises(hip.ArgumentError):
        cache.truncate(0, 21)
    cache.truncate(0, 8)
    assert cache.free_page_count() == 2
    cache.clear()
    assert cache.free_page_count() == 4 and cache.len(1) == 0
    cache.close()


def test_tensors_over_a_cache_keep_its_memory(hip, torch):
    ctx = _ctx(hip, torch, 2, 1, 64)
    for dtype in TYPES:
        cache = hip.PagedKVCache(ctx, 700, 16, 3, 5, dtype=dtype, layers=2)
        cache.map_rows(_ints(torch, [20]), *(torch.empty(20, dtype=torch.int32, device="cuda") for _ in range(3)))
        k, table, lens = cache.pages(1)[0], cache.table, cache.lens
        k.fill_(2.5)
        cache.close()
        del cache
        hip.PagedKVCache(ctx, 700, 16, 3, 5, dtype=dtype, layers=2)  # would come to lie there
        assert (k == 2.5).all() and table[0, :2].tolist() == [0, 1] and lens.tolist() == [20, 0, 0]
    closed = hip.PagedKVCache(ctx, 7, 16, 3, 5)
    closed.close()
    closed.close()
    with pytest.raises(hip.ArgumentError):
        closed.clear()


def test_a_table_of_angles_is_not_extended_while_recording(hip, torch):
    stream = torch.cuda.Stream()
    ctx = hip.AttnContext(2, 1, 64, max_positions=16)
    ctx.set_stream(stream.cuda_stream)
    cache = hip.PagedKVCache(ctx, 40, 64, 2, 40)
    x = [torch.ones((2, w * 64), device="cuda") for w in (2, 1, 1)]
    out = torch.zeros((2, 128), device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        torch.add(out, 0, out=out)  # (something to record)
        with pytest.raises(hip.ArgumentError, match="recorded"):
            ctx.step_paged(cache, *x, out)
    graph.replay()
    ctx.step_paged(cache, *x, out)
    ctx.sync()
    assert torch.allclose(out, torch.ones_like(out))


@pytest.mark.parametrize("dtype,P", [("bf16", 16), ("f32", 64), ("f16", 1024)])
def test_pages_behind_four_gigabytes(hip, torch, dtype, P):
    """Sequences in the last pages of pools of more than 2^32 bytes each, by every call."""
    H, KV, hd = 8, 4, 128
    rng = np.random.default_rng(6)
    ctx = _ctx(hip, torch, H, KV, hd)
    page = KV * P * hd * (4 if dtype == "f32" else 2)
    n_pages = (2 ** 32 + 2 ** 26) // page
    cache = hip.PagedKVCache(ctx, n_pages, P, 2, 40, dtype=dtype)
    cache.free_pages.copy_(torch.arange(n_pages, dtype=torch.int32, device="cuda"))  # the last page goes first
    plain = hip.KVCache(ctx, 2, 600)
    worst = 0.0
    for new, ids in (([400, 33], [0, 1]), ([1, 9], [1, 0]), ([1], [0])):
        rows = [torch.from_numpy(rng.standard_normal((sum(new), w * hd)).astype(np.float32)).cuda() for w in (H, KV, KV)]
        got = ctx.forward_paged(cache, *rows, new, seq_ids=ids)
        want = ctx.forward(plain, *rows, new, seq_ids=ids)
        ctx.sync()
        worst = max(worst, (got - want).abs().max().item())
    assert (cache.table[0, :pages_of(400, P)] >= n_pages - 40).all() and cache.table[0, 0].item() == n_pages - 1
    assert worst <= _tolerance(dtype)
    rows = [torch.from_numpy(rng.standard_normal((2, w * hd)).astype(np.float32)).cuda() for w in (H, KV, KV)]
    got = ctx.step_paged(cache, *rows, torch.empty_like(rows[0]))
    want = ctx.forward(plain, *rows, [1, 1])
    ctx.sync()
    assert (got - want).abs().max().item() <= _tolerance(dtype)
    cache.lengths_from_device()
    for a, b in zip(cache.read(0, 3, 0, cache.len(0)), plain.read(0, 3, 0, plain.len(0))):
        assert np.abs(a - b).max() <= (0 if dtype == "f32" else 2.0 ** -8 * np.abs(b).max())


def test_other_layers_use_the_rows_of_layer_0_only(hip, torch):
    H, KV, hd = 4, 2, 64
    ctx = _ctx(hip, torch, H, KV, hd)
    cache = hip.PagedKVCache(ctx, 20, 8, 3, 5, layers=2)
    rows = lambda n: [torch.zeros((n, w * hd), device="cuda") for w in (H, KV, KV)]  # noqa: E731
    lists = [torch.empty(3, dtype=torch.int32, device="cuda") for _ in range(3)]
    out = torch.empty((2, H * hd), device="cuda")
    steps = lambda layer: ctx.step_paged(cache, *rows(2), out, layer=layer)  # noqa: E731
    forward = lambda layer: ctx.forward_paged(cache, *rows(3), [2, 1], seq_ids=[2, 0], layer=layer)  # noqa: E731
    changes = (lambda: cache.map_rows(_ints(torch, [1]), *lists), lambda: cache.truncate(0, 0), lambda: cache.clear(),
               lambda: cache.clear(0))
    for change in changes:
        for call, other in ((steps, forward), (forward, steps)):
            cache.clear()
            call(0)
            call(1)
            cache.lengths_from_device()
            call(1)  # (nothing was changed)
            change()
            cache.lengths_from_device()
            with pytest.raises(hip.ArgumentError, match="layer"):
                call(1)
            cache.clear()
            call(0)
            cache.lengths_from_device()
            with pytest.raises(hip.ArgumentError, match="layer"):
                other(1)
    cache.clear()
    steps(0)
    with pytest.raises(hip.ArgumentError, match="layer"):
        ctx.step_paged(cache, *rows(1), out[:1], layer=1)


@pytest.mark.parametrize("dtype", TYPES)
def test_outputs_may_take_the_place_of_queries(hip, torch, dtype):
    H, KV, hd, P = 20, 1, 96, 16
    rng = np.random.default_rng(31)
    ctx = _ctx(hip, torch, H, KV, hd)
    lens = [9000, 3, 0, 700]
    cache, held = _filled(hip, torch, ctx, lens, P, dtype, rng)
    q = rng.standard_normal((4, H * hd)).astype(np.float32)
    seqs, positions = list(range(4)), [n - 1 for n in lens]
    t = torch.from_numpy(q).cuda()
    ctx.attend_paged(cache, _ints(torch, seqs), _ints(torch, positions), t, out=t)
    ctx.sync()
    _check_rows(t.cpu().numpy(), q, held, seqs, positions, hd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", ["q", "k", "v"])
def test_what_is_no_number_stays_in_its_row(hip, torch, what, dtype):
    """NaN in a query, or in a key or value that counts, makes NaN of the outputs it enters and of no others."""
    H, KV, hd, P = 4, 2, 64, 16
    rng = np.random.default_rng(2)
    ctx = _ctx(hip, torch, H, KV, hd)
    cache, held = _filled(hip, torch, ctx, [300, 300], P, dtype, rng)
    q = torch.from_numpy(rng.standard_normal((2, H * hd)).astype(np.float32)).cuda()
    args = _ints(torch, [0, 1]), _ints(torch, [299, 299])
    before = ctx.attend_paged(cache, *args, q)
    if what == "q":
        q[0, 2 * hd + 5] = float("nan")     # query head 2
        bad = torch.zeros_like(before, dtype=torch.bool)
        bad[0, 2 * hd:3 * hd] = True
    else:
        page = cache.table[0, 3].item()
        (cache.k if what == "k" else cache.v)[page, 1, 7, 9] = float("nan")  # kv head 1: query heads 2 and 3
        bad = torch.zeros_like(before, dtype=torch.bool)
        bad[0, 2 * hd:] = True
        if what == "v":
            bad[0] = False
            bad[0, 2 * hd + 9] = bad[0, 3 * hd + 9] = True
    after = ctx.attend_paged(cache, *args, q)
    ctx.sync()
    assert torch.equal(torch.isnan(after), bad)
    assert torch.equal(after[~bad], before[~bad])


def test_steps_on_another_stream(hip, torch):
    """A context moved to another stream takes its cache along; rows made there are seen there."""
    H, KV, hd = 4, 2, 64
    rng = np.random.default_rng(9)
    ctx = _ctx(hip, torch, H, KV, hd)
    cache, plain = hip.PagedKVCache(ctx, 40, 8, 3, 10, dtype="f32"), hip.KVCache(ctx, 3, 80)
    for turn in range(6):
        stream = torch.cuda.Stream()
        ctx.set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            rows = [torch.from_numpy(rng.standard_normal((3, w * hd)).astype(np.float32)).cuda(non_blocking=True) for w in (H, KV, KV)]
            got = ctx.step_paged(cache, *rows, torch.empty_like(rows[0]))
            want = ctx.forward(plain, *rows, [1, 1, 1])
            assert (got - want).abs().max().item() <= 2e-5, turn
    cache.lengths_from_device()
    assert [cache.len(s) for s in range(3)] == [6, 6, 6]
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)


# ---- recordings, and what the host knows ------------------------------------------------------------

def _rows(torch, rng, n, H, KV, hd):
    return [torch.from_numpy(rng.standard_normal((n, w * hd)).astype(np.float32)).cuda() for w in (H, KV, KV)]


def test_a_recorded_step_outlives_the_table_of_angles(hip, torch):
    """A longer table of angles, made for another cache, leaves recordings the one that they read."""
    H, KV, hd = 4, 2, 64
    rng = np.random.default_rng(11)
    stream = torch.cuda.Stream()
    ctx = hip.AttnContext(H, KV, hd, max_positions=64)
    ctx.set_stream(stream.cuda_stream)
    caches = [hip.PagedKVCache(ctx, 16, 8, 2, 8, dtype="f32") for _ in range(2)]
    x = _rows(torch, rng, 2, H, KV, hd)
    outs = [torch.zeros_like(x[0]) for _ in caches]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.step_paged(caches[0], *x, outs[0])
    for turn in range(4):
        if turn == 2:
            longer = hip.PagedKVCache(ctx, 64, 64, 1, 64)
            ctx.step_paged(longer, *(t[:1].contiguous() for t in x), torch.empty_like(x[0][:1]))
            ctx.sync()
            waste = [torch.full((64 * 32 * 2,), float("nan"), device="cuda") for _ in range(64)]
        for t in x:
            t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32)))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.step_paged(caches[1], *x, outs[1])
        ctx.sync()
        assert torch.equal(*outs), turn
    del waste


def test_a_table_wider_than_the_pool(hip, torch):
    """Sequences may be as wide as 2^30 rows where the pool holds a few thousand: angles are made for those."""
    H, KV, hd = 4, 2, 64
    rng = np.random.default_rng(12)
    ctx = _ctx(hip, torch, H, KV, hd)
    cache, plain = hip.PagedKVCache(ctx, 4, 1024, 1, 2 ** 20 - 1, dtype="f32"), hip.KVCache(ctx, 1, 4096)
    for n in (1500, 1, 3, 2000, 1):
        x = _rows(torch, rng, n, H, KV, hd)
        got, want = ctx.forward_paged(cache, *x, [n]), ctx.forward(plain, *x, [n])
        assert (got - want).abs().max().item() <= 2e-5, n
    with pytest.raises(hip.HipError, match="pages wanted"):
        ctx.forward_paged(cache, *_rows(torch, rng, 592, H, KV, hd), [592])
    x = _rows(torch, rng, 1, H, KV, hd)
    got = ctx.step_paged(cache, *x, torch.empty_like(x[0]))
    assert (got - ctx.forward(plain, *x, [1])).abs().max().item() <= 2e-5
    ctx.sync()
    one = _ints(torch, [0])
    with pytest.raises(hip.HipError, match="GiB"):  # of lists of the caller's own nothing is known
        ctx.append_paged(cache, one, one, *x, torch.empty_like(x[0]))


def test_calls_that_are_not_recorded(hip, torch):
    H, KV, hd = 4, 2, 64
    rng = np.random.default_rng(13)
    stream = torch.cuda.Stream()
    ctx = hip.AttnContext(H, KV, hd)
    ctx.set_stream(stream.cuda_stream)
    cache = hip.PagedKVCache(ctx, 16, 8, 2, 8)
    x = _rows(torch, rng, 12, H, KV, hd)
    ctx.forward_paged(cache, *x, [9, 3])
    out = torch.zeros_like(x[0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        torch.add(out, 1, out=out)
        for call in (lambda: cache.truncate(0, 3), lambda: cache.truncate(0, 9), lambda: cache.clear(), lambda: cache.clear(1),
                     lambda: cache.read(0, 0, 0, 3), cache.lengths_from_device, lambda: hip.PagedKVCache(ctx, 16, 8, 2, 8),
                     lambda: ctx.forward_paged(cache, *x, [9, 3])):
            with pytest.raises(hip.ArgumentError, match="recorded"):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 1).all() and cache.len(0) == 9 and cache.lens.tolist() == [9, 3] and cache.free_page_count() == 13
    cache.truncate(0, 3)
    assert cache.len(0) == 3
    ctx.sync()
    assert cache.lens.tolist() == [3, 3]


@pytest.mark.parametrize("new", [[1, 2], [20, 1]])
def test_lengths_that_the_host_missed(hip, torch, new):
    """Replays that the host does not see: what it plans on its own lengths changes nothing and is reported."""
    H, KV, hd = 4, 2, 64
    rng = np.random.default_rng(14)
    stream = torch.cuda.Stream()
    ctx = hip.AttnContext(H, KV, hd)
    ctx.set_stream(stream.cuda_stream)
    cache, plain = hip.PagedKVCache(ctx, 32, 8, 2, 16, dtype="f32"), hip.KVCache(ctx, 2, 128)
    x, more = _rows(torch, rng, 2, H, KV, hd), _rows(torch, rng, sum(new), H, KV, hd)
    out = torch.zeros_like(x[0])
    ctx.step_paged(cache, *x, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.step_paged(cache, *x, out)
    cache.lengths_from_device()
    for turn in range(3):
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.forward(plain, *x, [1, 1])
    ctx.forward(plain, *x, [1, 1])
    ctx.sync()
    assert cache.len(0) == 1 and cache.lens.tolist() == [4, 4]
    before = [t.clone() for t in (cache.table, cache.free_pages, cache.n_free, cache.k, cache.v)]
    for call in (lambda: cache.truncate(1, 0), lambda: ctx.forward_paged(cache, *more, new)):
        call()
        with pytest.raises(hip.ArgumentError, match="did not know"):
            ctx.sync()
        assert cache.lens.tolist() == [4, 4]
        for a, b in zip(before, (cache.table, cache.free_pages, cache.n_free, cache.k, cache.v)):
            assert torch.equal(a, b)
    cache.lengths_from_device()
    assert [cache.len(s) for s in range(2)] == [4, 4]
    got, want = ctx.forward_paged(cache, *more, new), ctx.forward(plain, *more, new)
    ctx.sync()
    assert (got - want).abs().max().item() <= 2e-5


@pytest.mark.parametrize("seq_pages", [20000, 40000])
def test_maps_of_many_pages(hip, torch, seq_pages):
    """Pages by the ten thousand, in one workgroup and in many; a step of a large pool."""
    n_pages, P = 70000, 8
    cache, model = hip.PagedKVCache(_ctx(hip, torch, 1, 1, 8), n_pages, P, 3, seq_pages), Pages(n_pages, P, 3, seq_pages)
    lists = [torch.empty(400000, dtype=torch.int32, device="cuda") for _ in range(3)]
    few = [torch.empty(3, dtype=torch.int32, device="cuda") for _ in range(3)]
    for entries, rows in (([(2, 150001), (0, 80003), (1, 160000)], lists), ([(1, -159999), (2, -1), (0, 3)], few), ([(0, -80006)], None),
                          ([(2, 1), (1, -1), (0, 1)], few), ([(2, -150001), (0, -1)], None), ([(0, 160000)], lists)):
        want = model.map(entries, rows[0].numel() if rows else 0)
        cache.map_rows(_ints(torch, [d for _, d in entries]), *(rows or ()), seq_ids=_ints(torch, [s for s, _ in entries]))
        cache.lengths_from_device()
        _same_state(cache, model, len(model.free))
        if rows:
            got = np.stack([t[:len(want)].cpu().numpy() for t in rows], 1)
            assert np.array_equal(got, np.array(want).reshape(-1, 3))
            assert all((t[len(want):] == -1).all() for t in rows)


def test_more_keys_than_can_be_counted(hip, torch):
    """Tables wide enough for 2^30 keys: so many rows of so many kv heads in one call are refused."""
    ctx = _ctx(hip, torch, 1024, 1024, 8)
    cache = hip.PagedKVCache(ctx, 1, 1024, 1, 2 ** 20 - 1)
    q = torch.zeros((16, 1024 * 8), device="cuda")
    rows = torch.zeros(16, dtype=torch.int32, device="cuda")
    for n in (16, 15, 5):
        with pytest.raises(hip.ArgumentError, match="2\\^42"):
            ctx.attend_paged(cache, rows[:n], rows[:n], q[:n])
    out = ctx.attend_paged(cache, rows[:3], rows[:3], q[:3])
    ctx.sync()
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd,n,rows", [(8, 8, 64, 16, 16), (16, 8, 128, 31, 31), (8, 8, 64, 39, 39), (16, 8, 96, 64, 64), (8, 8, 72, 65, 65), (8, 4, 128, 20, 200),
                                            (4, 2, 256, 30, 90)])
def test_spans_of_uneven_sequences(hip, torch, H, KV, hd, n, rows, dtype):
    """Lengths from nothing to some thousand keys: spans that begin and end anywhere, at pairs' ends, behind short ones, within one."""
    rng = np.random.default_rng(1000 * n + hd)
    ctx = _ctx(hip, torch, H, KV, hd)
    for turn in range(3):
        lens = np.exp(rng.uniform(0, np.log((300, 1200, 4000)[turn]), n)).astype(int) - (rng.random(n) < 0.1)
        cache, held = _filled(hip, torch, ctx, lens.tolist(), 16, dtype, rng, poison=float("nan"))
        q = rng.standard_normal((rows, H * hd)).astype(np.float32)
        seqs = (np.arange(rows) % n).tolist()
        positions = [int(lens[s]) - 1 - int(rng.integers(0, 3)) * (r >= n) for r, s in enumerate(seqs)]
        got = ctx.attend_paged(cache, _ints(torch, seqs), _ints(torch, positions), torch.from_numpy(q).cuda())
        ctx.sync()
        _check_rows(got.cpu().numpy(), q, held, seqs, [max(p, -1) for p in positions], hd)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("P", [8, 32])
def test_maps_of_more_rows_than_threads(hip, torch, P, shift):
    """Entries of no rows, of a few and of hundreds next to each other, in lists that begin on 16 bytes or do not."""
    rng = np.random.default_rng(P)
    n, room = 4096, 480001
    cache, model = hip.PagedKVCache(_ctx(hip, torch, 1, 1, 8), 60000, P, n, 80), Pages(60000, P, n, 80)
    for turn in range(3):
        entries = [(s, min(int(d), 80 * P - model.lens[s])) for s, d in
                   zip(rng.permutation(n).tolist(), rng.choice([0, 1, 2, 3, 5, 9, 70, 150, -2, -40], n))]
        entries = [(s, max(d, -model.lens[s])) for s, d in entries]
        lists = [torch.full((room + shift,), -7, dtype=torch.int32, device="cuda")[shift:] for _ in range(3)]
        want = np.full((room, 3), -1)
        rows = model.map(entries, room)
        want[:len(rows)] = rows
        cache.map_rows(_ints(torch, [d for _, d in entries]), *lists, seq_ids=_ints(torch, [s for s, _ in entries]))
        cache.lengths_from_device()
        _same_state(cache, model, len(model.free))
        assert np.array_equal(np.stack([t.cpu().numpy() for t in lists], 1), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd,rows", [(8, 8, 128, 44), (16, 8, 96, 45), (8, 8, 80, 47), (8, 8, 64, 150)])
def test_long_spans_of_many_pairs(hip, torch, H, KV, hd, rows, dtype):
    """Where half of the workgroups leave: rows by the dozen that share a few long sequences, and some that have next to nothing."""
    rng = np.random.default_rng(rows)
    ctx = _ctx(hip, torch, H, KV, hd)
    lens = [2100, 3990, 3000, 2777, 5]
    cache, held = _filled(hip, torch, ctx, lens, 32, dtype, rng, poison=float("nan"))
    seqs = [r % 4 for r in range(rows)]
    positions = [lens[s] - 1 - r for r, s in enumerate(seqs)]
    seqs[7], positions[7] = 4, 4
    seqs[9], positions[9] = 2, -1
    q = rng.standard_normal((rows, H * hd)).astype(np.float32)
    args = _ints(torch, seqs), _ints(torch, positions), torch.from_numpy(q).cuda()
    got = ctx.attend_paged(cache, *args)
    again = ctx.attend_paged(cache, *args)
    ctx.sync()
    _check_rows(got.cpu().numpy(), q, held, seqs, positions, hd)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 64, 65, 1000])
def test_rows_of_which_none_has_a_key(hip, torch, rows, dtype):
    ctx = _ctx(hip, torch, 8, 2, 64)
    cache = hip.PagedKVCache(ctx, 4, 8, 3, 2, dtype=dtype)
    q = torch.randn(rows, 512, device="cuda")
    seqs = [(0, 2, -1, 3)[r % 4] for r in range(rows)]
    out = torch.full_like(q, 7)
    for _ in range(2):
        ctx.attend_paged(cache, _ints(torch, seqs), _ints(torch, [-1 - r % 5 for r in range(rows)]), q, out)
    ctx.sync()
    for r, s in enumerate(seqs):
        assert (out[r] == (0 if s in (0, 2) else 7)).all(), r
