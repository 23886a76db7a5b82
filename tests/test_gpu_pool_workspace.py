"""The workspace of a pool's decode calls: what eager calls outgrow is freed, what
captured calls use stays, and growth takes no more than the call needs where
memory is short."""
import pytest
import torch

from gpu_util import dev_bf16, fast_kv, fast_q

pytestmark = pytest.mark.gpu

D, HKV, HQ, BLOCKS = 512, 2, 16, 64
GIB = 1 << 30


class Server:
    """A pool of one sequence's blocks, which every sequence of a batch shares: a
    batch of n needs n * BLOCKS * HQ * (D + 2) * 4 bytes of partials (one split a block)."""

    PER = BLOCKS * HQ * (D + 2) * 4

    def __init__(self, gpu):
        self.gpu = gpu
        self.pool = gpu.PagedPool(gpu.make_desc(HKV, D, 8), BLOCKS)
        n = BLOCKS * 16
        k, v = (dev_bf16(fast_kv(s, n, HKV, D))[None] for s in (1, 2))
        self.row = torch.arange(BLOCKS, dtype=torch.int32, device="cuda")[None]
        self.pool.append(k, v, self.row, torch.zeros(1, dtype=torch.int32, device="cuda"))
        self.q = dev_bf16(fast_q(3, 1, HQ, HKV, D))
        torch.cuda.synchronize()

    def args(self, n):
        """(q, tables, lengths, bound) of n sequences."""
        return (self.q.expand(n, HQ, D).contiguous(), self.row.expand(n, BLOCKS).contiguous(),
                self.row.new_full((n,), BLOCKS * 16), BLOCKS * 16)

    def run(self, args, windowed, out=None):
        if windowed:
            return self.pool.window_attention(*args, BLOCKS * 16, 0, 0.02, out=out)
        return self.pool.attention(*args, 0.02, out=out)

    def alone(self, args, windowed):
        """The call's result on a pool of its own."""
        other = Server(self.gpu)
        out = other.run(args, windowed)
        torch.cuda.synchronize()
        other.pool.close()
        return out


@pytest.fixture
def server(gpu):
    gpu.set_blocks_per_split(1)
    try:
        yield Server(gpu)
    finally:
        gpu.set_blocks_per_split(0)


def free():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("windowed", [True, False])
def test_eager_calls_keep_one_workspace(server, windowed):
    """Batches that grow a little each time: the pool holds the last one's partials."""
    sizes = [16, 18, 21, 24, 27, 31]
    calls = [(a, server.q.new_empty(a[0].shape), server.alone(a, windowed)) for a in map(server.args, sizes)]
    before = free()
    for a, out, want in calls:
        server.run(a, windowed, out=out)
        assert before - free() <= a[0].shape[0] * server.PER + (24 << 20)
        assert torch.equal(out, want)


@pytest.mark.parametrize("windowed", [True, False])
def test_captured_calls_keep_theirs(server, windowed):
    """Graphs of three sizes, each outgrown by the next and by eager calls: replays
    stay right, and all buffers together stay below three times the last."""
    sizes = (8, 9, 20)
    calls = [(a, server.alone(a, windowed)) for a in map(server.args, sizes)]
    eager = server.args(13)
    eager_want = server.alone(eager, windowed)
    before = free()
    graphs = []
    for n, (a, want) in zip(sizes, calls):
        out = torch.zeros_like(a[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            server.run(a, windowed, out=out)
        graphs.append((g, out, want))
        server.run(server.args(n + 1), windowed)
    server.run(server.args(40), windowed)
    assert before - free() <= 3 * 40 * server.PER + (128 << 20)  # (torch's own besides)
    for _ in range(3):
        for g, out, want in graphs:
            out.zero_()
            g.replay()
            assert torch.equal(server.run(eager, windowed), eager_want)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_growth_while_another_stream_captures(server):
    """An eager call outgrows the workspace inside another stream's capture: the
    capture survives, and the call's result is the usual one."""
    want = server.run(server.args(1), True)
    small, large = server.args(3), server.args(11)
    outs = [torch.zeros_like(a[0]) for a in (small, large)]
    server.run(small, True, out=outs[0])
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    eager, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        server.pool.window_attention(*large, BLOCKS * 16, 0, 0.02, out=outs[1], stream=eager)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert bool((outs[1] == want).all()) and bool((outs[0] == want).all()) and x.tolist() == [3.0] * 4


@pytest.mark.parametrize("captured", [False, True])
def test_growth_where_memory_is_short(server, captured):
    """A call a tenth larger than the one before, on a card that has no room for half
    as much again: eager calls need room for one workspace, captured ones for both."""
    n = 2 * GIB // server.PER
    want = server.run(server.args(1), True)
    small, large = server.args(n), server.args(n + n // 10)
    outs = [torch.zeros_like(a[0]) for a in (small, large)]
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            server.run(small, True, out=outs[0])
    else:
        server.run(small, True, out=outs[0])
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    # room left: 1 GiB (with the 2 that are freed: 3, of which 2.2 are needed), or
    # 2.75 GiB beside the workspace that is kept, less than half as much again (3)
    room = 11 * GIB // 4 if captured else GIB
    filler = []
    while free() > room + (64 << 20):
        filler.append(torch.empty(min(free() - room, 32 * GIB), dtype=torch.uint8, device="cuda"))
    try:
        server.run(large, True, out=outs[1])
        torch.cuda.synchronize()
    finally:
        del filler
        torch.cuda.empty_cache()
    assert bool((outs[1] == want).all())
    if captured:
        graph.replay()
        torch.cuda.synchronize()
    assert bool((outs[0] == want).all())
