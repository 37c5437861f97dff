"""Sequences that a caller made longer than the pool (pages that were dropped: table entries of no page), beyond the contexts' tables of angles."""
import numpy as np
import pytest

from paged_model import attended, turned
from test_gpu_paged import _ints, _rows, hip, torch  # noqa: F401

pytestmark = pytest.mark.gpu

H, KV, HD, P = 4, 2, 64, 8


class Far:
    """Sequence 0 has 2000 rows, of which the last 16 lie in pages; layer 0 and layer 1 have a context each."""

    def __init__(self, hip, torch, rng, positions=(0, 0), dtype="f32"):  # noqa: F811
        self.rng, self.torch = rng, torch
        self.ctxs = [hip.AttnContext(H, KV, HD, max_positions=n) for n in positions]
        for c in self.ctxs:
            c.set_stream(torch.cuda.current_stream().cuda_stream)
        self.cache = cache = hip.PagedKVCache(self.ctxs[0], 6, P, 2, 400, dtype=dtype, layers=2)
        for layer in range(2):
            for pool in cache.pages(layer):
                pool.copy_(torch.from_numpy(rng.standard_normal(pool.shape).astype(np.float32)))
        cache.table.fill_(-1)
        cache.table[0, 248:250] = _ints(torch, [4, 2])
        cache.lens.copy_(_ints(torch, [2000, 0]))
        cache.free_pages[:4] = _ints(torch, [0, 1, 3, 5])
        cache.n_free.fill_(4)
        torch.cuda.synchronize()

    def rows(self, n):
        return _rows(self.torch, self.rng, n, H, KV, HD)

    def check(self, layer, x, out, at):
        """Rows of sequence 0 at positions `at` are in the layer's pages, and the outputs are attention over what the pages have."""
        table = self.cache.table[0].cpu().numpy()
        pools = [t.float().cpu().numpy() for t in self.cache.pages(layer)]
        freq, positions = self.ctxs[layer].inv_freq(), np.array(at)
        q, k = (turned(t.cpu().numpy(), HD, positions, freq) for t in x[:2])
        out = out.cpu().numpy().reshape(len(at), H, HD)
        size = lambda t: np.abs(t).max()  # noqa: E731
        for r, pos in enumerate(at):
            page, row = table[pos // P], pos % P
            # (turned in float32: cos, sin, two products, a sum, each half a step of the pair's size)
            assert np.abs(pools[0][page, :, row].reshape(-1) - k[r]).max() <= 2.0 ** -24 * 10 * 2 * size(k[r])
            assert np.array_equal(pools[1][page, :, row].reshape(-1), x[2][r].cpu().numpy())
            keys = [t for t in range(pos + 1) if table[t // P] >= 0]
            held = [np.stack([pool[table[t // P], :, t % P] for t in keys], 1) for pool in pools]
            want, off = attended(q[r].reshape(H, HD), *held)
            # (queries turned in float32: 6 u of a pair's size in every score, which `attended` allows hd + 4 of)
            assert (np.abs(out[r] - want) <= 1.5 * off).all(), (layer, pos)


def test_steps_wait_until_the_host_knows(hip, torch):  # noqa: F811
    far = Far(hip, torch, np.random.default_rng(1))
    cache, zero = far.cache, _ints(torch, [0])
    out = torch.full((1, H * HD), 5.0, device="cuda")
    before = [t.clone() for layer in range(2) for t in cache.pages(layer)]
    for layer in range(2):
        far.ctxs[layer].step_paged(cache, *far.rows(1), out, seq_ids=zero, layer=layer)
    with pytest.raises(hip.HipError, match="cos/sin table"):
        far.ctxs[0].sync()
    far.ctxs[0].sync()
    assert (out == 5.0).all() and cache.lens.tolist() == [2000, 0] and cache.n_free.item() == 4
    assert all(torch.equal(a, b) for a, b in zip(before, [t for layer in range(2) for t in cache.pages(layer)]))
    cache.lengths_from_device()
    n = 2000
    for turn in range(3):
        for layer in range(2):
            x = far.rows(1)
            far.ctxs[layer].step_paged(cache, *x, out, seq_ids=zero, layer=layer)
            far.ctxs[0].sync()
            far.check(layer, x, out, [n])
        n += 1
    cache.lengths_from_device()
    assert cache.len(0) == n
    for layer in range(2):
        x = far.rows(8)
        got = far.ctxs[layer].forward_paged(cache, *x, [8], seq_ids=[0], layer=layer)
        far.ctxs[0].sync()
        far.check(layer, x, got, list(range(n, n + 8)))


def test_rows_of_a_call_that_the_host_plans(hip, torch):  # noqa: F811
    far = Far(hip, torch, np.random.default_rng(2))
    far.cache.lengths_from_device()
    for n, new in ((2000, 3), (2003, 1)):
        for layer in range(2):
            x = far.rows(new)
            got = far.ctxs[layer].forward_paged(far.cache, *x, [new], seq_ids=[0], layer=layer)
            far.ctxs[0].sync()
            far.check(layer, x, got, list(range(n, n + new)))


@pytest.mark.parametrize("mode", ["device", "host"])
@pytest.mark.parametrize("new", [9, 20])
def test_prompts_on_keys_of_no_page(hip, torch, new, mode):  # noqa: F811
    """More rows than are attended one by one: such keys would count as zeros there, and the call is reported; its rows can be taken back."""
    far = Far(hip, torch, np.random.default_rng(5))
    cache, ctx = far.cache, far.ctxs[0]
    cache.lengths_from_device()
    x = far.rows(new)
    with pytest.raises(hip.ArgumentError, match="no page of the pool"):
        if mode == "device":
            ctx.forward_paged(cache, *x, [new], seq_ids=[0])
            ctx.sync()
        else:
            ctx.forward_paged(cache, *(t.cpu().numpy() for t in x), [new], seq_ids=[0])
    assert cache.len(0) == 2000 + new and cache.lens.tolist() == [2000 + new, 0]
    cache.truncate(0, 2000)
    ctx.sync()
    assert cache.free_page_count() == 4
    got = ctx.forward_paged(cache, *(t[:8].contiguous() for t in x), [8], seq_ids=[0])
    ctx.sync()
    far.check(0, [t[:8] for t in x], got, list(range(2000, 2008)))
    # a sequence of pages of its own beside it
    y = far.rows(new)
    ctx.forward_paged(cache, *y, [new], seq_ids=[1])
    ctx.sync()


def test_a_layer_whose_table_of_angles_is_shorter(hip, torch):  # noqa: F811
    far = Far(hip, torch, np.random.default_rng(3), positions=(4000, 0))
    cache, zero = far.cache, _ints(torch, [0])
    outs = [torch.full((1, H * HD), 5.0, device="cuda") for _ in range(2)]
    x = far.rows(1)
    before = [t.clone() for t in cache.pages(1)]
    for layer in range(2):
        far.ctxs[layer].step_paged(cache, *x, outs[layer], seq_ids=zero, layer=layer)
    with pytest.raises(hip.HipError, match="cos/sin table"):
        far.ctxs[0].sync()
    far.check(0, x, outs[0], [2000])
    assert (outs[1] == 5.0).all() and all(torch.equal(a, b) for a, b in zip(before, cache.pages(1)))
    cache.lengths_from_device()
    for layer in range(2):
        far.ctxs[layer].step_paged(cache, *x, outs[layer], seq_ids=zero, layer=layer)
        far.ctxs[0].sync()
        far.check(layer, x, outs[layer], [2001])


def test_recorded_steps_have_the_table_that_they_were_recorded_with(hip, torch):  # noqa: F811
    """Replays beyond it find no room; what is recorded once the host knows the lengths goes on."""
    rng = np.random.default_rng(4)
    stream = torch.cuda.Stream()
    far = Far(hip, torch, rng)
    for c in far.ctxs:
        c.set_stream(stream.cuda_stream)
    cache, ctx = far.cache, far.ctxs[0]
    x, out = far.rows(1), torch.full((1, H * HD), 5.0, device="cuda")
    ids = _ints(torch, [0])
    graphs = []
    for known in (False, True):
        if known:
            cache.lengths_from_device()
            ctx.step_paged(cache, *x, out, seq_ids=_ints(torch, [1]))  # (extends the table, which no recording can)
            ctx.sync()
            out.fill_(5.0)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            ctx.step_paged(cache, *x, out, seq_ids=ids)
    n = 2000
    for turn in range(4):
        for known, graph in enumerate(graphs):
            for t in x:
                t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32)))
            out.fill_(5.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            if known:
                ctx.sync()
                far.check(0, x, out, [n])
                n += 1
            else:
                with pytest.raises(hip.HipError, match="cos/sin table"):
                    ctx.sync()
                assert (out == 5.0).all()
            assert cache.lens.tolist() == [n, 1]


def test_a_step_of_more_keys_than_can_be_counted(hip, torch):  # noqa: F811
    """Tables wide enough for 2^30 keys: a step of so many rows is refused before it maps one."""
    ctx = hip.AttnContext(1024, 1024, 8)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    cache = hip.PagedKVCache(ctx, 20, 1024, 16, 2 ** 20 - 1)
    x = [torch.ones((16, 1024 * 8), device="cuda") for _ in range(3)]
    out = torch.full_like(x[0], 5.0)
    for n in (16, 15, 5):
        with pytest.raises(hip.ArgumentError, match="2\\^42"):
            ctx.step_paged(cache, *(t[:n] for t in x), out[:n])
    assert cache.len(0) == 0 and cache.free_page_count() == 20  # (the host still knows)
    with pytest.raises(hip.ArgumentError, match="2\\^42"):
        ctx.forward_paged(cache, *(t[:5] for t in x), [1] * 5)
    cache.lengths_from_device()
    assert [cache.len(s) for s in range(16)] == [0] * 16 and cache.free_page_count() == 20
    ctx.step_paged(cache, *(t[:3] for t in x), out[:3])
    cache.lengths_from_device()
    assert [cache.len(s) for s in range(4)] == [1, 1, 1, 0] and (out[3:] == 5.0).all()
    assert ((out[:3] - 1).abs() <= 3.01 * 2.0 ** -24).all()  # (one key: its value, by two products and a quotient, each rounded)


@pytest.mark.parametrize("where", ["free pages", "table"])
def test_rows_that_have_no_page(hip, torch, where):  # noqa: F811
    """A free page, or the entry of a sequence's last page, that the pool does not have: the row is left alone and reported, others are not."""
    rng = np.random.default_rng(6)
    far = Far(hip, torch, rng, positions=(4000, 4000))
    cache, ctx = far.cache, far.ctxs[0]
    if where == "table":  # sequence 0 goes on within its last page
        cache.lens[0] = 1999
        cache.table[0, 249] = 77
    else:  # sequence 0 takes the first page
        cache.free_pages[3] = -3
    cache.lengths_from_device()
    for layer in range(2):
        x, out = far.rows(2), torch.full((2, H * HD), 5.0, device="cuda")
        far.ctxs[layer].step_paged(cache, *x, out, layer=layer)
        with pytest.raises(hip.ArgumentError, match="the pool does not have"):
            ctx.sync()
        assert (out[0] == 5.0).all()
        # (one key: its value, by two products and a quotient, each rounded)
        v = x[2][1].view(KV, 1, HD).expand(KV, H // KV, HD).reshape(-1)
        assert ((out[1] - v).abs() <= 3.01 * 2.0 ** -24 * v.abs()).all()
