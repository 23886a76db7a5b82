"""Attention of a paged pool over a window with sinks, several queries per
sequence, every cache mode against the oracle's stored rows in 64 bits."""
import numpy as np
import pytest

from gpu_util import dev_bf16, fast_kv
from window_util import AFFINE, CODEBOOK, PLAIN, Paged, check_window, queries, window_reference

pytestmark = pytest.mark.gpu

CONFIGS = [  # mode, D, bits, Hkv, Hq
    (AFFINE, 256, 4, 8, 16), (AFFINE, 512, 8, 2, 16), (AFFINE, 128, 4, 1, 3), (AFFINE, 256, 8, 2, 2),
    (CODEBOOK, 512, 3, 2, 16), (CODEBOOK, 256, 2, 4, 4), (CODEBOOK, 128, 4, 2, 10),
    (PLAIN, 512, 16, 2, 16), (PLAIN, 256, 16, 8, 16), (PLAIN, 128, 16, 1, 5),
]


def check(ora, p, out, q, start, window, sinks, scale, rows=None):
    for s, first in enumerate(start):
        for i in range(q.shape[1]) if rows is None else rows:
            ref = window_reference(ora, p.oracles[s], q[s, i], first + i, window, sinks, scale)
            check_window(out[s, i], ref, 6.0, f"sequence {s} row {i} position {first + i}")


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", CONFIGS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (16, 16), (33, 4), (60, 77), (5000, 3)])
def test_window_prefill(gpu, ora, mode, D, bits, Hkv, Hq, window, sinks):
    """45 queries after 0 .. 305 positions; hidden slots NaN, pages given back."""
    import torch

    start, n = [0, 1, 16, 100, 305], 45
    lens = [x + n for x in start]
    p = Paged(gpu, ora, mode, D, bits, Hkv, lens)
    p.hide(start, [x - 1 for x in lens], window, sinks)
    q = np.stack([queries(40 + s, n, Hq, Hkv, D) for s in range(len(start))])
    for dtype in (torch.float32, torch.bfloat16):
        out = p.pool.window_prefill(dev_bf16(q), p.table(), p.lens_dev(start), window, sinks, D ** -0.5,
                                    dtype=dtype)
        torch.cuda.synchronize()
        check(ora, p, out, q, start, window, sinks, D ** -0.5, rows=(0, 1, 15, 16, 17, 31, 32, 43, 44))


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", CONFIGS)
def test_window_prefill_step(gpu, ora, mode, D, bits, Hkv, Hq):
    """Chunks of 1, 7, 64 and 90 tokens appended and attended in one call."""
    import torch

    start, window, sinks = [0, 5, 64, 250], 50, 9
    p = Paged(gpu, ora, mode, D, bits, Hkv, start, room=170)
    for n in (1, 7, 64, 90):
        k, v = (np.stack([fast_kv(n * 31 + s + x, n, Hkv, D, outliers=False) for s in range(len(start))])
                for x in (0, 13))
        q = np.stack([queries(n + s, n, Hq, Hkv, D) for s in range(len(start))])
        out = p.pool.window_prefill_step(dev_bf16(k), dev_bf16(v), p.table(), p.lens_dev(start), dev_bf16(q),
                                         window, sinks, D ** -0.5, dtype=torch.float32)
        torch.cuda.synchronize()
        for s in range(len(start)):
            p.oracles[s].append(k[s], v[s])
        check(ora, p, out, q, start, window, sinks, D ** -0.5, rows={0, n // 2, n - 1})
        start = [x + n for x in start]


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", [CONFIGS[0], CONFIGS[1], CONFIGS[2], CONFIGS[4], CONFIGS[7], CONFIGS[9]])
@pytest.mark.parametrize("start", [[3000], [2100, 40]])
def test_window_prefill_split(gpu, ora, mode, D, bits, Hkv, Hq, start):
    """Few queries over a long window: split over the keys, the sinks' blocks in
    the first range, eager and (in the pool's workspace) captured."""
    import torch

    n, window, sinks = 5, 1500, 100
    lens = [x + n for x in start]
    p = Paged(gpu, ora, mode, D, bits, Hkv, lens)
    p.hide(start, [x - 1 for x in lens], window, sinks)
    q = np.stack([queries(4 + s, n, Hq, Hkv, D) for s in range(len(start))])
    qd, table, first = dev_bf16(q), p.table(), p.lens_dev(start)

    def call(out):
        return p.pool.window_prefill(qd, table, first, window, sinks, D ** -0.5, max_seq_len=max(lens), out=out)

    eager = call(torch.empty(qd.shape, dtype=torch.float32, device="cuda"))
    torch.cuda.synchronize()
    check(ora, p, eager, q, start, window, sinks, D ** -0.5)
    held = torch.zeros_like(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(held)
    for _ in range(3):
        held.zero_()
        graph.replay()
        call(torch.empty_like(eager))
        torch.cuda.synchronize()
        assert torch.equal(held, eager)


def test_one_query_is_the_decode_call(gpu, ora):
    """A chunk of one query and the single-token call agree."""
    import torch

    for mode, D, bits, Hkv, Hq in CONFIGS[:1] + CONFIGS[4:5] + CONFIGS[7:8]:
        lens = [700, 30]
        p = Paged(gpu, ora, mode, D, bits, Hkv, lens)
        q = dev_bf16(np.stack([queries(s, 1, Hq, Hkv, D) for s in range(2)]))
        a = p.pool.window_prefill(q, p.table(), p.lens_dev([n - 1 for n in lens]), 200, 20, 0.06,
                                  dtype=torch.float32)
        b = p.pool.window_attention(q[:, 0].contiguous(), p.table(), p.lens_dev(), 700, 200, 20, 0.06,
                                    dtype=torch.float32)
        torch.cuda.synchronize()
        check_window(a[:, 0], b.double().cpu().numpy(), 12.0)


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq,n", [(AFFINE, 512, 8, 2, 16, 333), (PLAIN, 128, 16, 4, 32, 600),
                                                  (CODEBOOK, 256, 3, 4, 32, 300), (AFFINE, 256, 4, 4, 32, 300)])
def test_window_prefill_tail(gpu, ora, mode, D, bits, Hkv, Hq, n):
    """More work-groups than run at once: the last ones' keys are split."""
    import torch

    start, window, sinks = [900, 1000, 40, 700], 1000, 21
    p = Paged(gpu, ora, mode, D, bits, Hkv, [x + n for x in start])
    q = np.stack([queries(4 + s, n, Hq, Hkv, D) for s in range(len(start))])
    qd, table, first = dev_bf16(q), p.table(), p.lens_dev(start)

    def call(out):
        return p.pool.window_prefill(qd, table, first, window, sinks, D ** -0.5, out=out)

    eager = call(torch.empty(qd.shape, dtype=torch.float32, device="cuda"))
    again = call(torch.empty(qd.shape, dtype=torch.float32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(eager, again)
    check(ora, p, eager, q, start, window, sinks, D ** -0.5, rows=(0, 1, n // 2, n - 9, n - 1))
    held = torch.zeros_like(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(held)
    for _ in range(3):
        held.zero_()
        graph.replay()
        call(again)
        torch.cuda.synchronize()
        assert torch.equal(held, eager) and torch.equal(again, eager)
