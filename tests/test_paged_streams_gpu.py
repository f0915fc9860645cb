"""paged_attention's split contexts on several streams at once and in graphs: a
graph's workspace is its own wherever it is replayed, grows with no call before the
capture, outlives other sizes, and is used again when the graph is gone."""
import numpy as np
import pytest

from gpu_util import lq
from paged_ref import Batch, cache_struct, random_cache

pytestmark = pytest.mark.gpu


class Call:
    """One sequence per context, a token each, 8 heads on 4."""

    def __init__(self, torch, seed, ctx, heads=8, hs=128, page=64):
        rng = np.random.default_rng(seed)
        batch = Batch(rng, [1] * len(ctx), ctx, page)
        codes, scales = random_cache(rng, batch.n_pages, 4, hs, page)
        self.keep = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), *batch.device(torch)
        self.cache, self.batch, self.heads = cache_struct(*self.keep[:2], 4, hs, page), self.keep[2], heads
        self.q = torch.from_numpy(rng.standard_normal((len(ctx), heads * hs)).astype(np.float32)).cuda()
        self.out, self.lse = torch.zeros_like(self.q), torch.zeros(len(ctx), heads, device="cuda")

    def __call__(self, out=None):
        out = self.out if out is None else out
        lq.paged_attention(out.data_ptr(), self.q.data_ptr(), self.heads, self.cache, self.batch, lse_ptr=self.lse.data_ptr())


@pytest.fixture
def streams(cuda):
    made = [cuda.cuda.Stream() for _ in range(3)]
    yield made
    cuda.cuda.synchronize()
    lq.set_stream(None)


def on(stream):
    lq.set_stream(stream.cuda_stream)


def graph_of(*calls):
    lq.graph_begin()
    for c in calls:
        c()
    return lq.graph_end()


def plain(torch, *calls):
    """Each call's bits, alone on its own."""
    out = []
    for c in calls:
        c()
        lq.sync()
        out.append((c.out.clone(), c.lse.clone()))
    return out


def test_capture_without_a_call_before(cuda, streams):
    torch = cuda
    small, large = Call(torch, 1, [3000]), Call(torch, 2, [2000, 1, 4000, 900])
    want = plain(torch, small, large)  # on another stream
    on(streams[0])
    g = graph_of(small, large, small)
    for _ in range(5):
        for c in (small, large):
            c.out.zero_(), c.lse.zero_()
        torch.cuda.synchronize()
        lq.graph_launch(g)
        lq.sync()
        for c, (out, lse) in zip((small, large), want):
            assert torch.equal(c.out, out) and torch.equal(c.lse, lse)
    lq.graph_destroy(g)


def test_capture_by_torch(cuda, streams):
    torch = cuda
    call = Call(torch, 3, [5000, 700])
    (out, lse), = plain(torch, call)
    on(streams[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=streams[1]):
        call()
    for _ in range(3):
        call.out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(call.out, out) and torch.equal(call.lse, lse)


def test_graphs_and_calls_at_once(cuda, streams):
    """Two graphs captured on one stream, replayed on two others while that stream
    makes calls of its own: everyone's bits are what they are alone."""
    torch = cuda
    calls = [Call(torch, i, ctx) for i, ctx in enumerate(([6000, 5000], [7000], [3000, 20, 4000]))]
    want = plain(torch, *calls)
    on(streams[0])
    graphs = [graph_of(*[c] * 8) for c in calls[:2]]
    for _ in range(30):
        for c in calls:
            c.out.zero_(), c.lse.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams[1:]):
            on(st)
            lq.graph_launch(g)
        on(streams[0])
        for _ in range(8):
            calls[2]()
        torch.cuda.synchronize()
        for c, (out, lse) in zip(calls, want):
            assert torch.equal(c.out, out) and torch.equal(c.lse, lse)
    lq.sync()
    for g in graphs:
        lq.graph_destroy(g)


def test_larger_calls_between_capture_and_replay(cuda, streams):
    torch = cuda
    small, large = Call(torch, 4, [2500]), Call(torch, 5, [3000] * 12, heads=64)
    want = plain(torch, small, large)
    on(streams[2])
    small()  # the stream's own workspace, of the least size
    g = graph_of(small)
    large()
    small.out.zero_()
    lq.graph_launch(g)
    large()
    lq.sync()
    for c, (out, lse) in zip((small, large), want):
        assert torch.equal(c.out, out) and torch.equal(c.lse, lse)
    lq.graph_destroy(g)


def test_workspaces_are_used_again(cuda, streams):
    """A hundred graphs made and destroyed one after another hold what a few do."""
    torch = cuda
    call = Call(torch, 6, [4000])
    (out, lse), = plain(torch, call)
    on(streams[0])
    free = None
    for i in range(100):
        g = graph_of(call)
        lq.graph_launch(g)
        lq.sync()
        lq.graph_destroy(g)
        torch.cuda.synchronize()
        if i == 10:
            free = torch.cuda.mem_get_info()[0]
    assert torch.equal(call.out, out)
    # a workspace is 1 MB or more: ninety of them would show
    assert free - torch.cuda.mem_get_info()[0] < 32 << 20
