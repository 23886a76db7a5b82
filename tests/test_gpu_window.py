"""Attention of a paged pool over a window with sinks, one token per sequence:
position p sees j <= p with j > p - window or j < sinks. Every cache mode against
the oracle's stored rows in 64 bits; hidden slots hold NaNs and infinities and
pages without visible slots are given back (their table entries lead nowhere)."""
import numpy as np
import pytest

import synth
from gpu_util import check_attention, check_codes, dev_bf16, fast_kv, kv_batch
from window_util import AFFINE, CODEBOOK, PLAIN, Paged, check_window, queries, window_reference

pytestmark = pytest.mark.gpu

CONFIGS = [  # mode, D, bits, Hkv, Hq
    (AFFINE, 256, 4, 8, 16), (AFFINE, 256, 4, 2, 12), (AFFINE, 512, 8, 2, 16), (AFFINE, 128, 4, 1, 3),
    (AFFINE, 128, 8, 4, 8), (AFFINE, 256, 8, 2, 2), (AFFINE, 512, 4, 1, 8),
    (CODEBOOK, 512, 3, 2, 16), (CODEBOOK, 256, 2, 4, 4), (CODEBOOK, 128, 4, 2, 10), (CODEBOOK, 256, 3, 1, 7),
    (PLAIN, 512, 16, 2, 16), (PLAIN, 256, 16, 8, 16), (PLAIN, 128, 16, 1, 5),
]
# lengths: none, one, block ends, inside and past the window
LENS = [0, 1, 15, 16, 17, 33, 64, 65, 100, 257, 400]


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", CONFIGS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 16), (33, 4), (48, 17), (100, 130), (5000, 0)])
def test_window_attention(gpu, ora, mode, D, bits, Hkv, Hq, window, sinks):
    import torch

    p = Paged(gpu, ora, mode, D, bits, Hkv, LENS)
    p.hide([n - 1 for n in LENS], [n - 1 for n in LENS], window, sinks)
    q = np.stack([queries(900 + s, 1, Hq, Hkv, D)[0] for s in range(len(LENS))])
    scale = D ** -0.5
    for dtype in (torch.float32, torch.bfloat16):
        out = p.pool.window_attention(dev_bf16(q), p.table(), p.lens_dev(), max(LENS), window, sinks, scale,
                                      dtype=dtype)
        torch.cuda.synchronize()
        for s, n in enumerate(LENS):
            ref = window_reference(ora, p.oracles[s], q[s], n - 1, window, sinks, scale)
            check_window(out[s], ref, 6.0, f"{dtype} length {n}")


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", [CONFIGS[0], CONFIGS[1], CONFIGS[2], CONFIGS[3], CONFIGS[7], CONFIGS[11]])
@pytest.mark.parametrize("bps", [0, 1, 3, 8, 9])
def test_window_attention_splits(gpu, ora, mode, D, bits, Hkv, Hq, bps):
    """Splits that start and end inside the sinks' blocks and the window, the
    streams of single waves (8 blocks and more) and of wave pairs, lengths on
    both sides of the first gap."""
    import torch

    lens, window, sinks = [1000, 613, 352, 351, 350, 340, 20], 301, 43
    p = Paged(gpu, ora, mode, D, bits, Hkv, lens)
    p.hide([n - 1 for n in lens], [n - 1 for n in lens], window, sinks)
    q = np.stack([queries(70 + s, 1, Hq, Hkv, D)[0] for s in range(len(lens))])
    gpu.set_blocks_per_split(bps)
    try:
        out = p.pool.window_attention(dev_bf16(q), p.table(), p.lens_dev(), max(lens), window, sinks,
                                      D ** -0.5, dtype=torch.float32)
        torch.cuda.synchronize()
    finally:
        gpu.set_blocks_per_split(0)
    for s, n in enumerate(lens):
        ref = window_reference(ora, p.oracles[s], q[s], n - 1, window, sinks, D ** -0.5)
        check_window(out[s], ref, 6.0, f"length {n}")


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", CONFIGS)
def test_window_decode_step(gpu, ora, mode, D, bits, Hkv, Hq):
    """Three steps of ragged sequences (an empty one among them): outputs, the
    stored codes, and every other slot as it was."""
    import torch

    lens, window, sinks = [0, 1, 31, 32, 130, 300], 40, 5
    p = Paged(gpu, ora, mode, D, bits, Hkv, lens, room=3)
    before = p.pool.storage().clone()
    for step in range(3):
        k, v = (np.stack([fast_kv(500 + 50 * step + s + x, 1, Hkv, D, outliers=False) for s in range(len(lens))])
                for x in (0, 25))
        now = [n + step for n in lens]
        q = np.stack([queries(300 + 10 * step + s, 1, Hq, Hkv, D)[0] for s in range(len(lens))])
        out = p.pool.window_decode_step(dev_bf16(k), dev_bf16(v), p.table(), p.lens_dev(now),
                                        p.lens_dev([n + 1 for n in now]), max(now) + 1, dev_bf16(q), window,
                                        sinks, D ** -0.5, dtype=torch.float32)
        torch.cuda.synchronize()
        for s, n in enumerate(now):
            p.oracles[s].append(k[s], v[s])
            ref = window_reference(ora, p.oracles[s], q[s], n, window, sinks, D ** -0.5)
            check_window(out[s], ref, 6.0, f"step {step} position {n}")
    codes, meta = p.pool.read_codes()
    torch.cuda.synchronize()
    for s, n in enumerate(lens):
        pos = np.arange(n + 3)
        slots = p.tables[s, pos // 16].astype(np.int64) * 16 + pos % 16
        idx = torch.from_numpy(slots).cuda()

        class Stored:
            codes, meta = p.oracles[s].codes[:n + 3], p.oracles[s].meta[:n + 3]

        check_codes(codes[idx], meta[idx], Stored, what=f"sequence {s}")
    for b in p.spare:
        assert torch.equal(p.pool.storage()[int(b)], before[int(b)])


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", [CONFIGS[0], CONFIGS[8], CONFIGS[12]])
def test_window_wider_than_the_sequences(gpu, ora, mode, D, bits, Hkv, Hq):
    """A window that hides nothing is the pool's plain attention (which needs
    unwritten slots as a new pool has them)."""
    import torch

    lens = [3, 200, 77]
    p = Paged(gpu, ora, mode, D, bits, Hkv, lens)
    q = dev_bf16(np.stack([queries(5 + s, 1, Hq, Hkv, D)[0] for s in range(3)]))
    clean = Paged(gpu, ora, mode, D, bits, Hkv, lens, dirty=False)
    args = (q, p.table(), p.lens_dev(), max(lens))
    for window, sinks in ((200, 0), (1 << 30, 1 << 30), (150, 50)):
        out = p.pool.window_attention(*args, window, sinks, 0.05, dtype=torch.float32)
        want = clean.pool.attention(*args, 0.05, dtype=torch.float32)
        torch.cuda.synchronize()
        check_window(out, want.double().cpu().numpy(), 6.0, f"window {window}")


def test_window_attention_bad_pages(gpu, ora):
    """Table entries outside the pool in visible places read some block of the
    pool (no fault); other sequences' outputs are theirs alone."""
    import torch

    mode, D, bits, Hkv, Hq = CONFIGS[0]
    lens, window, sinks = [200, 200], 64, 4
    p = Paged(gpu, ora, mode, D, bits, Hkv, lens)
    q = np.stack([queries(5 + s, 1, Hq, Hkv, D)[0] for s in range(2)])
    p.tables[0, -2:] = [-7, p.n_blocks + 100]
    p.tables[0, 0] = 2 ** 31 - 1
    out = p.pool.window_attention(dev_bf16(q), p.table(), p.lens_dev(), 200, window, sinks, 0.05,
                                  dtype=torch.float32)
    torch.cuda.synchronize()
    check_window(out[1], window_reference(ora, p.oracles[1], q[1], 199, window, sinks, 0.05), 6.0)


def test_window_step_of_a_padded_batch(gpu, ora):
    """Rows of length 0 (and below) write no slot and get zeros; an empty batch is
    no call."""
    import torch

    mode, D, bits, Hkv, Hq = CONFIGS[0]
    p = Paged(gpu, ora, mode, D, bits, Hkv, [50, 40, 30], room=2)
    before = p.pool.storage().clone()
    k, v = (dev_bf16(fast_kv(s, 3, Hkv, D, outliers=False))[:, None].contiguous() for s in (1, 2))
    q = queries(3, 3, Hq, Hkv, D)
    out = p.pool.window_decode_step(k, v, p.table(), p.lens_dev([50, -1, -6]), p.lens_dev([51, 0, -5]), 51,
                                    dev_bf16(q), 20, 3, 0.06, dtype=torch.float32)
    torch.cuda.synchronize()
    p.oracles[0].append(fast_kv(1, 3, Hkv, D, outliers=False)[:1], fast_kv(2, 3, Hkv, D, outliers=False)[:1])
    check_window(out[0], window_reference(ora, p.oracles[0], q[0], 50, 20, 3, 0.06), 6.0)
    assert bool((out[1:] == 0).all())
    blocks = torch.arange(p.n_blocks) != int(p.tables[0, 50 // 16])
    assert torch.equal(p.pool.storage()[blocks], before[blocks])
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    empty = p.pool.window_attention(torch.zeros((0, Hq, D), dtype=torch.bfloat16, device="cuda"),
                                    torch.zeros((0, 4), dtype=torch.int32, device="cuda"), none, 64, 20)
    assert empty.shape == (0, Hq, D)


def test_window_first_call_captured_and_other_stream(gpu, ora):
    """A capture that is a pool's first call allocates its workspace; a stream
    given to the call is the one it runs on."""
    import torch

    mode, D, bits, Hkv, Hq = CONFIGS[2]
    lens = [900, 333]
    p = Paged(gpu, ora, mode, D, bits, Hkv, lens)
    q = dev_bf16(np.stack([queries(5 + s, 1, Hq, Hkv, D)[0] for s in range(2)]))
    table, n = p.table(), p.lens_dev()
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.pool.window_attention(q, table, n, 900, 500, 4, 0.05, out=out)
    side = torch.cuda.Stream()
    for _ in range(3):
        out.zero_()
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        want = p.pool.window_attention(q, table, n, 900, 500, 4, 0.05, stream=side)
        side.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", [CONFIGS[2], CONFIGS[7], CONFIGS[11]])
def test_pages_past_4_gib(gpu, ora, mode, D, bits, Hkv, Hq):
    """A pool of more than 4 GiB whose last pages hold the sequence: attention, a
    chunk, copied blocks and kept tokens as in a small pool."""
    import torch

    n, window, sinks = 150, 60, 5
    small = Paged(gpu, ora, mode, D, bits, Hkv, [n], spare=40, dirty=False)
    size = small.pool.storage()[0].numel()
    big = gpu.PagedPool(gpu.make_desc(Hkv, D, bits, mode=mode), (9 << 29) // size + 64)
    off = big.n_blocks - small.n_blocks
    big.storage()[off:].copy_(small.pool.storage())
    q = dev_bf16(queries(3, 4, Hq, Hkv, D))
    keep = torch.arange(0, n, 3, dtype=torch.int32, device="cuda")[None]
    count = torch.tensor([keep.shape[1]], dtype=torch.int32, device="cuda")
    spare = torch.from_numpy(small.spare.astype(np.int32)).cuda()
    outs = []
    for pool, base in ((small.pool, 0), (big, off)):
        table = small.table() + base
        one = pool.window_attention(q[:1], table, small.lens_dev(), n, window, sinks, 0.05)
        four = pool.window_prefill(q[None], table, small.lens_dev([n - 4]), window, sinks, 0.05)
        gpu.copy_blocks([pool], table[0, :4].contiguous(), spare[:4] + base)
        dst = (spare[8:8 + 4] + base)[None].contiguous()
        pool.compact(table, keep, count, dst)
        full = pool.window_attention(q[:1], dst, count, 64, 1000, 0, 0.05)
        moved = pool.window_attention(q[:1], (spare[:4] + base)[None].contiguous(), small.lens_dev([64]), 64, 1000, 0,
                                      0.05)
        outs.append((one, four, full, moved))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert torch.equal(small.pool.storage(), big.storage()[off:])


def test_window_step_graph(gpu, ora):
    """A captured step replayed as its inputs change, with eager calls between
    that need a larger workspace and with another stream: bit for bit the eager
    result each time."""
    import torch

    mode, D, bits, Hkv, Hq = CONFIGS[0]
    lens, window, sinks = [900, 500, 700], 400, 4
    p = Paged(gpu, ora, mode, D, bits, Hkv, lens, room=64)
    table = p.table()
    k, v = (torch.zeros((3, 1, Hkv, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros((3, Hq, D), dtype=torch.bfloat16, device="cuda")
    start, now, out = p.lens_dev(), p.lens_dev([n + 1 for n in lens]), torch.empty_like(q)

    def step(o):
        return p.pool.window_decode_step(k, v, table, start, now, 964, q, window, sinks, 0.06, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    for i in range(4):
        for x, s in ((k, 1), (v, 2)):
            x.copy_(dev_bf16(fast_kv(60 * i + s, 3, Hkv, D, outliers=False))[:, None])
        q.copy_(dev_bf16(queries(9 + i, 3, Hq, Hkv, D)))
        graph.replay()
        got = out.clone()
        want = step(torch.empty_like(q))
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {i}"
        start += 1
        now += 1
        if i == 1:  # a batch that outgrows the workspace that the graph uses
            big = dev_bf16(queries(3, 24, Hq, Hkv, D))
            p.pool.window_attention(big, table[:1].repeat(24, 1), now[:1].repeat(24), 964, 900, 4, 0.06)


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", CONFIGS)
@pytest.mark.parametrize("scale", [1.0, 0.02])
def test_window_of_outlier_channels(gpu, ora, mode, D, bits, Hkv, Hq, scale):
    """K, V and q with channels 20 times the others, at the model's scale and a
    soft one, both calls: within the 2e-2 that every attention of the library
    holds (before a bf16 output's own rounding)."""
    import torch

    n, chunk, window, sinks = 230, 7, 70, 9
    p = Paged(gpu, ora, mode, D, bits, Hkv, [0], room=n)
    k, v = kv_batch(1, n, Hkv, D), kv_batch(2, n, Hkv, D)
    p.oracles[0].append(k, v)
    p.pool.append(dev_bf16(k[None]), dev_bf16(v[None]), p.table(), p.lens_dev([0]))
    q = synth.q_rows(3, Hq, Hkv, D, synth.outlier_channels(1, Hkv, D), batch=chunk)
    for dtype in (torch.float32, torch.bfloat16):
        some = p.pool.window_prefill(dev_bf16(q[None]), p.table(), p.lens_dev([n - chunk]), window, sinks, scale,
                                     dtype=dtype)
        one = p.pool.window_attention(dev_bf16(q[-1:]), p.table(), p.lens_dev([n]), n, window, sinks, scale,
                                      dtype=dtype)
        torch.cuda.synchronize()
        ref = np.stack([window_reference(ora, p.oracles[0], q[i], n - chunk + i, window, sinks, scale)
                        for i in range(chunk)])
        check_attention(some[0], ref, f"{dtype} chunk")
        check_attention(one, ref[-1:], f"{dtype} token")
