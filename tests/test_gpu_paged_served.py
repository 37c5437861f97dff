"""Requests served from pages, each output against the definition in 64 bits over the rows that the pages hold: a row lost, misplaced or seen
by another request shows in pages of every type, whatever their rounding."""
import numpy as np
import pytest

from paged_model import attended, pages_of, turned
from test_gpu_paged import TYPES, _ctx, _ints, _rows, hip, torch  # noqa: F401

pytestmark = pytest.mark.gpu

HALF = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


class Served:
    """What each sequence was given, and what it must have and get back."""

    def __init__(self, torch, ctx, cache, norms, freq):  # noqa: F811
        self.torch, self.ctx, self.cache, self.norms, self.freq = torch, ctx, cache, norms, freq
        self.given = {}

    def check(self, entries, q, k, v, out):
        hd, KV, H = self.ctx.head_dim, self.ctx.num_kv_heads, self.ctx.num_heads
        q, k, v, out = (t.cpu().numpy() for t in (q, k, v, out))
        u, at = 2.0 ** -24, 0
        steps = (hd / 2 + 16 if self.norms[0] is not None else 10) * 2
        for s, n in entries:
            old = self.given.get(s, (np.zeros((0, KV * hd)),) * 2)
            had, rows = len(old[0]), slice(at, at + n)
            positions = np.arange(had, had + n)
            mine = turned(q[rows], hd, positions, self.freq, self.norms[0]).reshape(n, H, hd)
            keys = np.concatenate([old[0], turned(k[rows], hd, positions, self.freq, self.norms[1])])
            values = np.concatenate([old[1], v[rows]])
            self.given[s] = keys, values
            held = [self.cache.read(s, c, 0, had + n) for c in range(KV)]
            hk, hv = (np.stack([h[i] for h in held]) for i in range(2))
            # The pages' rows: values rounded once; keys after the half steps of norm and rotation, of a row's largest number (as in the test
            # of placing), and then rounded once.
            assert np.array_equal(hv, self.torch.from_numpy(values.astype(np.float32)).to(self.cache.k.dtype).float().numpy().reshape(had + n, KV, hd).transpose(1, 0, 2))
            exact = keys.reshape(had + n, KV, hd).transpose(1, 0, 2)
            off = u * steps * np.abs(exact).max(-1, keepdims=True)
            assert (np.abs(hk - exact) <= off + HALF[self.cache.dtype] * (np.abs(exact) + off) + 2.0 ** -25).all(), s
            # Outputs over those rows: a float32 computation's bound, and what queries that are off by as much as keys may do to a score
            for r in range(n):
                seen = had + r + 1
                want, bound = attended(mine[r], hk[:, :seen], hv[:, :seen])
                per = lambda x: x.repeat(H // KV)[:, None]  # noqa: E731  (of a kv head, for each of its query heads)
                moved = u * steps * np.abs(mine[r]).max(-1, keepdims=True) * per(np.abs(hk[:, :seen]).sum(-1).max(-1)) / np.sqrt(hd)
                bound = 2 * bound + 2 * moved * per(np.abs(hv[:, :seen]).max((1, 2)))
                assert (np.abs(out[at + r].reshape(H, hd) - want) <= bound).all(), (s, r, np.abs(out[at + r].reshape(H, hd) - want).max(), bound.min())
                assert np.median(bound) < 3e-3  # (one key of 300 weighs more)
            at += n


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd,P", [(8, 2, 64, 16), (5, 5, 80, 8), (6, 2, 128, 32)])
def test_requests_that_come_and_go(hip, torch, H, KV, hd, P, dtype, norm):  # noqa: F811
    rng = np.random.default_rng(H * hd + norm)
    norms = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) if norm else None for _ in range(2)]
    ctx = _ctx(hip, torch, H, KV, hd, q_norm=norms[0], k_norm=norms[1])
    slots = 4
    cache = hip.PagedKVCache(ctx, 4 * pages_of(280, P), P, slots, pages_of(280, P), dtype=dtype)
    served, live = Served(torch, ctx, cache, norms, ctx.inv_freq()), {}
    for turn in range(20):
        entries = []
        for s in rng.permutation(slots).tolist():
            if s not in live:
                entries.append((s, int(rng.choice([1, 2, 8, 9, 17, 40, 130]))))
            elif rng.random() < 0.2 or live[s] > 250:
                cache.clear(s)
                served.given.pop(s)
                del live[s]
            else:
                entries.append((s, int(rng.choice([1, 1, 3, 8, 20]))))
        if turn % 3 == 0:
            entries = [(s, 1) for s, _ in entries]
        if not entries:
            continue
        q, k, v = _rows(torch, rng, sum(n for _, n in entries), H, KV, hd)
        if turn % 3 == 0:
            out = ctx.step_paged(cache, q, k, v, torch.full_like(q, 3.0), seq_ids=_ints(torch, [s for s, _ in entries]))
            cache.lengths_from_device()
        else:
            out = ctx.forward_paged(cache, q, k, v, [n for _, n in entries], seq_ids=[s for s, _ in entries])
            ctx.sync()
        served.check(entries, q, k, v, out)
        for s, n in entries:
            live[s] = live.get(s, 0) + n
            assert cache.len(s) == live[s]


@pytest.mark.parametrize("dtype,P", [("bf16", 16), ("f32", 64), ("f16", 1024), ("f16", 8)])
def test_requests_behind_four_gigabytes(hip, torch, dtype, P):  # noqa: F811
    """Pages on both sides of 2^32 bytes of a pool, the last one among them, in an order of no order."""
    H, KV, hd = 8, 4, 128
    rng = np.random.default_rng(P)
    ctx = _ctx(hip, torch, H, KV, hd)
    page = KV * P * hd * (4 if dtype == "f32" else 2)
    n_pages = (2 ** 32 + 2 ** 26) // page
    cache = hip.PagedKVCache(ctx, n_pages, P, 2, pages_of(600, P), dtype=dtype)
    want = 2 * cache.seq_pages
    edge = [n_pages - 1, 2 ** 32 // page - 1, 2 ** 32 // page, 2 ** 32 // page + 1]
    order = np.concatenate([np.setdiff1d(rng.permutation(n_pages)[:want + 4], edge)[:want], rng.permutation(edge)])
    rest = np.setdiff1d(np.arange(n_pages), order)
    cache.free_pages.copy_(torch.from_numpy(np.concatenate([rest, order]).astype(np.int32)))
    served = Served(torch, ctx, cache, (None, None), ctx.inv_freq())
    for new, ids in (([300, 33], [0, 1]), ([1, 9], [1, 0]), ([7], [0]), (None, None), ([1], [0])):
        entries = list(zip(ids, new)) if new else [(0, 1), (1, 1)]
        q, k, v = _rows(torch, rng, sum(n for _, n in entries), H, KV, hd)
        if new:
            out = ctx.forward_paged(cache, q, k, v, new, seq_ids=ids)
        else:
            out = ctx.step_paged(cache, q, k, v, torch.empty_like(q))
        cache.lengths_from_device()
        served.check(entries, q, k, v, out)
    held = set(cache.table[0, :pages_of(cache.len(0), P)].tolist()) | set(cache.table[1, :pages_of(cache.len(1), P)].tolist())
    assert set(edge[:min(len(edge), len(held))]) & held
