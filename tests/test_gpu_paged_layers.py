"""Layers behind the first place the rows that layer 0 mapped, or none: maps that come between, seen by the host or not."""
import numpy as np
import pytest

from paged_model import attended
from test_gpu_paged import _ints, _rows, hip, torch  # noqa: F401

pytestmark = pytest.mark.gpu

H, KV, HD, P = 4, 2, 64, 8


class Two:
    """Two layers of one cache on a stream of their own, and a recorded call that changes lengths."""

    def __init__(self, hip, torch, rng, dtype="f32"):  # noqa: F811
        self.torch, self.stream = torch, torch.cuda.Stream()
        self.ctx = hip.AttnContext(H, KV, HD)
        self.ctx.set_stream(self.stream.cuda_stream)
        self.cache = hip.PagedKVCache(self.ctx, 20, P, 3, 5, dtype=dtype, layers=2)
        self.lists = [torch.empty(40, dtype=torch.int32, device="cuda") for _ in range(3)]
        self.x = _rows(torch, rng, 12, H, KV, HD)
        self.out = torch.full_like(self.x[0], 5.0)
        torch.cuda.synchronize()
        self.ctx.forward_paged(self.cache, *(t[:2].contiguous() for t in self.x), [2], seq_ids=[1])
        self.ctx.sync()

    def record(self, call):
        graph = self.torch.cuda.CUDAGraph()
        self.torch.cuda.synchronize()
        with self.torch.cuda.graph(graph, stream=self.stream):
            call()
        self.cache.lengths_from_device()
        return graph

    def replay(self, graph):
        with self.torch.cuda.stream(self.stream):
            graph.replay()

    def step(self, layer):
        n = 3
        self.ctx.step_paged(self.cache, *(t[:n] for t in self.x), self.out[:n], layer=layer)

    def forward(self, new, layer):
        n = sum(new)
        self.ctx.forward_paged(self.cache, *(t[:n] for t in self.x), new, seq_ids=[2, 0], out=self.out[:n], layer=layer)

    def pages(self):
        self.ctx.sync()
        return [t.clone() for t in self.cache.pages(1)]


KINDS = ["step", "few rows", "many rows"]


def _call(two, kind):
    return {"step": two.step, "few rows": lambda layer: two.forward([2, 1], layer), "many rows": lambda layer: two.forward([9, 3], layer)}[kind]


@pytest.mark.parametrize("fetched", [True, False])
@pytest.mark.parametrize("kind", KINDS)
def test_a_replayed_map_between_the_layers(hip, torch, kind, fetched):  # noqa: F811
    """Requests end and others begin, with as many rows, in a replay: layer 1 of the rows before it places nothing, and is refused by the host
    once it can know (of a step it cannot: a replay may have mapped new rows by then)."""
    two = Two(hip, torch, np.random.default_rng(1))
    drop, admit = _ints(torch, [-100] * 3), _ints(torch, [0] * 3)

    def change():  # (the changes are in device memory)
        two.cache.map_rows(drop)
        two.cache.map_rows(admit, *two.lists, seq_ids=order)

    order = _ints(torch, [0, 1, 2])
    graph = two.record(change)
    call = _call(two, kind)
    call(0)
    two.cache.lengths_from_device()
    lens = two.cache.lens.clone()
    drop.copy_(-lens)
    order.copy_(_ints(torch, [2, 0, 1]))
    admit.copy_(lens[order.long()])
    torch.cuda.synchronize()
    before = two.pages()
    two.out.fill_(5.0)
    torch.cuda.synchronize()
    two.replay(graph)
    two.ctx.sync()
    assert torch.equal(two.cache.lens, lens)
    if fetched:
        two.cache.lengths_from_device()
    if fetched and kind != "step":
        with pytest.raises(hip.ArgumentError, match="other rows than layer 0"):
            call(1)
        two.ctx.sync()
    else:
        call(1)
        with pytest.raises(hip.ArgumentError, match="after layer 0 mapped"):
            two.ctx.sync()
        two.ctx.sync()  # said once
    for a, b in zip(before, two.pages()):
        assert torch.equal(a, b)
    if fetched or kind != "many rows":
        assert (two.out == 5.0).all()
    # (and the pass begins anew)
    two.cache.lengths_from_device()
    call(0)
    call(1)
    two.ctx.sync()


@pytest.mark.parametrize("what", ["table", "lens", "shorter"])
@pytest.mark.parametrize("kind", KINDS)
def test_a_caller_that_writes_between_the_layers(hip, torch, kind, what):  # noqa: F811
    """A page of a sequence is replaced, or its length changed, through the arrays: layer 1 is refused once the host was told."""
    two = Two(hip, torch, np.random.default_rng(2))
    call = _call(two, kind)
    call(0)
    two.cache.lengths_from_device()
    if what == "table":
        two.cache.table[2, 0] = 19  # (nobody's)
    else:
        two.cache.lens[2] = 0 if what == "shorter" else two.cache.len(2) + 1
    torch.cuda.synchronize()
    before = two.pages()
    two.cache.lengths_from_device()
    with pytest.raises(hip.ArgumentError, match="layer 0"):
        call(1)
        two.ctx.sync()
    for a, b in zip(before, two.pages()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fetched", [True, False])
def test_a_layer_recorded_by_itself(hip, torch, fetched):  # noqa: F811
    """Layer 0 replayed, the layer behind it eager or a recording of its own: it has the rows of the last replay."""
    rng = np.random.default_rng(3)
    two = Two(hip, torch, rng)
    first = two.record(lambda: two.step(0))
    second = two.record(lambda: two.step(1))
    lens = [0, 2, 0]
    for turn in range(6):
        for t in two.x:
            t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32)))
        torch.cuda.synchronize()
        two.replay(first)
        if fetched and turn != 3:
            two.cache.lengths_from_device()
        if turn == 3:
            two.step(1)  # eager
        else:
            two.replay(second)
        two.cache.lengths_from_device()
        lens = [n + 1 for n in lens]
        assert [two.cache.len(s) for s in range(3)] == lens
        v = two.x[2][:3].cpu().numpy().reshape(3, KV, HD)
        for s in range(3):
            for c in range(KV):
                assert np.array_equal(two.cache.read(s, c, lens[s] - 1, 1, layer=1)[1][0], v[s, c])
                assert two.cache.read(s, c, 0, lens[s], layer=1)[0].any(1)[2 if s == 1 else 0:].all()  # (sequence 1's first two have none there)
    q_rows = two.out[:3].cpu().numpy()
    assert np.isfinite(q_rows).all() and not (q_rows == 5.0).any()


def test_a_step_without_room_in_every_layer(hip, torch):  # noqa: F811
    two = Two(hip, torch, np.random.default_rng(4))
    two.cache.map_rows(_ints(torch, [40, 38, 40]), *[torch.empty(118, dtype=torch.int32, device="cuda") for _ in range(3)])
    two.ctx.sync()
    before = two.pages()
    two.step(0)
    two.step(1)
    with pytest.raises(hip.HipError, match="free pages"):
        two.ctx.sync()
    two.ctx.sync()
    assert (two.out == 5.0).all()
    for a, b in zip(before, two.pages()):
        assert torch.equal(a, b)
    two.cache.lengths_from_device()
    assert [two.cache.len(s) for s in range(3)] == [40, 40, 40]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layers_of_a_step_against_the_definition(hip, torch, dtype):  # noqa: F811
    """Steps of two layers over prompts, lengths fetched between the layers or not: outputs of each layer over the rows read back."""
    rng = np.random.default_rng(5)
    two = Two(hip, torch, rng, dtype)
    for layer in range(2):
        two.forward([9, 3], layer)
    freq = two.ctx.inv_freq()
    for turn in range(4):
        outs = []
        for layer in range(2):
            two.step(layer)
            if turn % 2:
                two.cache.lengths_from_device()
            two.ctx.sync()
            outs.append(two.out[:3].cpu().numpy().reshape(3, H, HD))
        two.cache.lengths_from_device()
        for layer in range(2):
            for s in (0, 2):
                n = two.cache.len(s)
                rows = [two.cache.read(s, c, 0, n, layer=layer) for c in range(KV)]
                k, v = (np.stack([r[i] for r in rows]) for i in range(2))
                x = two.x[0][s].cpu().numpy().reshape(H, HD).astype(np.float64)
                angle = (np.float32(n - 1) * freq).astype(np.float64)
                a, b = x[:, :HD // 2], x[:, HD // 2:]
                turned = np.concatenate([a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)], 1)
                want, off = attended(turned, k, v)
                # (queries turned in float32 are off by 6 u of a pair's size at most, in every score, which `attended` allows hd + 4 of)
                assert (np.abs(outs[layer][s] - want) <= 1.5 * off).all(), (turn, layer, s)


def test_a_call_without_memory_leaves_the_rows_of_the_one_before(hip, torch):  # noqa: F811
    """400 GB of gathered rows are not to be had: the call changes nothing, and the last one's other layers go on."""
    rng = np.random.default_rng(6)
    heads, hd = 2048, 8
    ctx = hip.AttnContext(heads, heads, hd)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    cache = hip.PagedKVCache(ctx, 4, 1024, 2, 3100, layers=2)
    cache.table[1].fill_(-1)  # (a long sequence whose pages were dropped)
    cache.lens[1] = 3_000_000
    cache.lengths_from_device()
    x = _rows(torch, rng, 3, heads, heads, hd)
    ctx.forward_paged(cache, *x, [3], seq_ids=[0])
    ctx.sync()
    with pytest.raises(hip.HipError, match="hipMalloc"):
        ctx.forward_paged(cache, *_rows(torch, rng, 400, heads, heads, hd), [400], seq_ids=[1])
    assert (cache.len(0), cache.len(1), cache.free_page_count()) == (3, 3_000_000, 3)
    got = ctx.forward_paged(cache, *x, [3], seq_ids=[0], layer=1)
    ctx.sync()
    assert cache.lens.tolist() == [3, 3_000_000] and cache.n_free.item() == 3
    v = x[2].view(3, heads, hd).to(torch.bfloat16)
    page = cache.table[0, 0].item()
    assert torch.equal(cache.pages(1)[1][page, :, :3], v.transpose(0, 1))
    # (one key: its value, w v (1 / w) for a weight w near 1; the first product, the quotient and the second product are rounded by half
    # a step, 2^-24, each)
    want = v[0].float().flatten()
    assert ((got[0] - want).abs() <= 3.01 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("rows", [8192, 8193, 70000])
@pytest.mark.parametrize("where", [None, "first", "last", "middle"])
def test_a_caller_that_writes_to_the_table_of_prompts(hip, torch, rows, where):  # noqa: F811
    """Rows enough for a look by many workgroups: a page of one of two sequences is replaced, or none."""
    ctx = hip.AttnContext(1, 1, 8)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    some = rows // 3
    cache = hip.PagedKVCache(ctx, rows // 16 + 4, 16, 2, rows // 16 + 2, layers=2)
    x = [torch.ones((rows, 8), device="cuda") for _ in range(3)]
    forward = lambda layer: ctx.forward_paged(cache, *x, [some, rows - some], layer=layer)  # noqa: E731
    forward(0)
    if where == "first":
        cache.table[0, 0] = cache.n_pages - 1
    elif where == "last":
        cache.table[1, (rows - some - 1) // 16] = cache.n_pages - 1
    elif where == "middle":
        cache.table[1, rows // 64] = cache.n_pages - 1
    cache.lengths_from_device()
    if where:
        before = [t.clone() for t in cache.pages(1)]
        with pytest.raises(hip.ArgumentError, match="layer 0"):
            forward(1)
        assert all(torch.equal(a, b) for a, b in zip(before, cache.pages(1)))
    else:
        out = forward(1)
        ctx.sync()
        # (values of 1: the outputs' numerator and the weights' sum are sums of as many numbers, each off by rows half steps at most)
        assert ((out - 1).abs() <= (2 * rows + 40) * 2.0 ** -24).all()
        assert (cache.pages(1)[1][cache.table[1, 0], :, :16] == 1).all()
