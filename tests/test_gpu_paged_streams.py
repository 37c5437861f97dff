"""Outputs that the paged calls make themselves, where the context works on another stream than torch's current one."""
import numpy as np
import pytest

from test_gpu_paged import _ints, hip, torch  # noqa: F401

pytestmark = pytest.mark.gpu

H, KV, HD, P, N = 8, 2, 64, 16, 32
LONG = 20_000_000  # clock ticks: milliseconds at least


class Side:
    """A context and cache on a stream; `call(name)` makes one of the calls without a place for its output."""

    def __init__(self, hip, torch, stream):  # noqa: F811
        rng = np.random.default_rng(1)
        self.ctx = hip.AttnContext(H, KV, HD)
        self.ctx.set_stream(stream.cuda_stream)
        self.cache = hip.PagedKVCache(self.ctx, 40, P, 4, 10, dtype="f32")
        self.x = [torch.from_numpy(rng.standard_normal((N, w * HD)).astype(np.float32)).cuda() for w in (H, KV, KV)]
        self.lists = [torch.empty(N, dtype=torch.int32, device="cuda") for _ in range(3)]
        self.cache.map_rows(_ints(torch, [N]), *self.lists)
        self.ctx.sync()
        self.ctx.append_paged(self.cache, *self.lists[:2], *self.x, q_rot=torch.empty_like(self.x[0]))
        self.cache.lengths_from_device()
        torch.cuda.synchronize()

    def call(self, name):
        if name == "append":
            return self.ctx.append_paged(self.cache, *self.lists[:2], *self.x)
        if name == "attend":
            return self.ctx.attend_paged(self.cache, self.lists[2], self.lists[1], self.x[0])
        return self.ctx.forward_paged(self.cache, *self.x, [N], seq_ids=[1])


CALLS = ["append", "attend", "forward"]


@pytest.mark.parametrize("name", CALLS)
def test_memory_that_the_current_stream_still_uses(hip, torch, name):  # noqa: F811
    other = torch.cuda.Stream()
    want = Side(hip, torch, torch.cuda.current_stream()).call(name)
    side = Side(hip, torch, other)
    torch.cuda.synchronize()
    old = torch.empty((N, H * HD), device="cuda")
    torch.cuda._sleep(LONG)
    old.fill_(float("nan"))
    at = old.data_ptr()
    del old
    got = side.call(name)
    assert got.data_ptr() == at  # (the memory of the one before, which is written last otherwise)
    side.ctx.sync()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", CALLS)
def test_memory_that_goes_back_before_it_is_written(hip, torch, name):  # noqa: F811
    other = torch.cuda.Stream()
    side = Side(hip, torch, other)
    side.call(name)  # (what a call allocates the first time)
    if name == "forward":
        side.cache.clear(1)
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        torch.cuda._sleep(LONG)
    got = side.call(name)
    at = got.data_ptr()
    del got
    new = torch.zeros((N, H * HD), device="cuda")
    assert new.data_ptr() == at
    torch.cuda.synchronize()
    assert (new == 0).all()


@pytest.mark.parametrize("name", CALLS)
def test_outputs_are_there_for_the_current_stream(hip, torch, name):  # noqa: F811
    other = torch.cuda.Stream()
    want = Side(hip, torch, torch.cuda.current_stream()).call(name)
    side = Side(hip, torch, other)
    with torch.cuda.stream(other):
        torch.cuda._sleep(LONG)
    got = side.call(name) + 0.0  # (no wait in between)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", CALLS)
def test_a_context_on_the_default_stream(hip, torch, name):  # noqa: F811
    want = Side(hip, torch, torch.cuda.current_stream()).call(name)
    side = Side(hip, torch, torch.cuda.default_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda._sleep(LONG)
        got = side.call(name) + 0.0
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", ["append", "attend"])
def test_outputs_made_while_the_current_stream_is_recorded(hip, torch, name):  # noqa: F811
    """The context's stream takes part in the recording by the waits, and leaves it by them."""
    here, other = torch.cuda.Stream(), torch.cuda.Stream()
    side = Side(hip, torch, other)
    want = side.call(name)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=here):
        got = side.call(name)
        twice = got + got
    for turn in range(4):
        got.fill_(float("nan"))
        twice.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(here):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(twice, want + want), turn
        side.x[1].add_(0.0)
    del graph
