"""Blocks of pools copied, and sequences compacted to the tokens they keep: bit
for bit, every other slot as it was, in every cache mode."""
import numpy as np
import pytest

import synth
from window_util import AFFINE, CODEBOOK, PLAIN, Paged, check_window, queries, window_reference
from gpu_util import dev_bf16, fast_kv

pytestmark = pytest.mark.gpu

MODES = [  # mode, D, bits, Hkv
    (AFFINE, 128, 4, 3), (AFFINE, 256, 4, 8), (AFFINE, 512, 4, 1), (AFFINE, 128, 8, 2), (AFFINE, 256, 8, 1),
    (AFFINE, 512, 8, 2), (CODEBOOK, 128, 2, 2), (CODEBOOK, 128, 3, 1), (CODEBOOK, 256, 3, 3),
    (CODEBOOK, 512, 3, 2), (CODEBOOK, 512, 2, 1), (CODEBOOK, 256, 4, 2), (PLAIN, 128, 16, 1), (PLAIN, 256, 16, 3),
    (PLAIN, 512, 16, 2),
]


def i32(x):
    import torch

    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def filled(gpu, mode, D, bits, Hkv, n_blocks, seed=3):
    """A pool of random bytes."""
    import torch

    pool = gpu.PagedPool(gpu.make_desc(Hkv, D, bits, mode=mode), n_blocks)
    g = torch.Generator().manual_seed(seed)
    st = pool.storage()
    st.copy_(torch.randint(0, 256, st.shape, generator=g, dtype=torch.uint8))
    return pool


@pytest.mark.parametrize("mode,D,bits,Hkv", MODES)
@pytest.mark.parametrize("n", [0, 1, 9, 200])
def test_copy_blocks(gpu, mode, D, bits, Hkv, n):
    import torch

    pool = filled(gpu, mode, D, bits, Hkv, 2 * n + 5)
    order = np.argsort(synth.splitmix64(5, 2 * n + 5))
    src, dst = order[:n], order[n:2 * n]
    want = pool.storage().clone()
    want[torch.from_numpy(dst)] = want[torch.from_numpy(src)]
    gpu.copy_blocks([pool], i32(src), i32(dst))
    torch.cuda.synchronize()
    assert torch.equal(pool.storage(), want)


def test_copy_blocks_of_many_pools(gpu):
    """70 pools of different layouts and sizes in one call; pairs that do not fit
    a pool, or copy a block to itself, are left out there; one source for two
    destinations."""
    import torch

    pools = [filled(gpu, *MODES[i % len(MODES)], 6 + i % 4, seed=i) for i in range(70)]
    src, dst = [0, 0, 7, 3, -1, 3, 5, 2 ** 31 - 1], [1, 4, 2, 8, 2, 3, -9, 0]
    want = [p.storage().clone() for p in pools]
    for w in want:
        for a, b in zip(src, dst):
            if 0 <= a < len(w) and 0 <= b < len(w):
                w[b] = w[a]
    gpu.copy_blocks(pools, i32(src), i32(dst))
    torch.cuda.synchronize()
    for p, w in zip(pools, want):
        assert torch.equal(p.storage(), w)


def test_copy_blocks_of_more_threads_than_a_grid_holds(gpu):
    """Blocks of 512 KB in a list of 131080 pairs, nearly all of which name no block:
    over 2^32 threads."""
    import torch

    pool = filled(gpu, PLAIN, 512, 16, 16, 9)
    n = 131080
    src, dst = np.full(n, -1, np.int32), np.zeros(n, np.int32)
    at = [0, 131070, 131071, n - 1]
    src[at], dst[at] = [0, 1, 2, 3], [4, 5, 6, 7]
    want = pool.storage().clone()
    want[4:8] = want[0:4]
    gpu.copy_blocks([pool], i32(src), i32(dst))
    torch.cuda.synchronize()
    assert torch.equal(pool.storage(), want)


def test_compact_of_more_threads_than_a_grid_holds_is_refused(gpu):
    import torch

    pool = filled(gpu, *MODES[0], 8)
    before = pool.storage().clone()
    t, n = i32([[0, 1]]), i32([2])
    assert gpu.load_library().fmkv_paged_compact(pool._h, t.data_ptr(), 2, t.data_ptr(), 1 << 28, n.data_ptr(),
                                                 t.data_ptr(), 1 << 24, 1, None) == gpu.FMKV_ERR_INVALID_ARG
    torch.cuda.synchronize()
    assert torch.equal(pool.storage(), before)


def test_copy_blocks_graph_and_stream(gpu):
    import torch

    pool = filled(gpu, *MODES[1], 12)
    src, dst = i32([1, 2]), i32([8, 9])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu.copy_blocks([pool], src, dst)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.copy_blocks([pool], src, dst)
    for a in ([1, 2], [3, 0], [5, 5]):
        src.copy_(i32(a))
        want = pool.storage().clone()
        want[8], want[9] = want[a[0]], want[a[1]]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool.storage(), want)


def slots(table, pos):
    return table[pos // 16].astype(np.int64) * 16 + pos % 16


@pytest.mark.parametrize("mode,D,bits,Hkv", MODES)
def test_compact(gpu, mode, D, bits, Hkv):
    """Ragged sequences that keep everything, nothing, one token, every third, a
    reversed and a repeated selection."""
    import torch

    lens = [33, 200, 16, 75, 131, 64, 50]
    need = [-(-n // 16) for n in lens]
    n_blocks = 2 * sum(need) + 3
    pool = filled(gpu, mode, D, bits, Hkv, n_blocks)
    order = np.argsort(synth.splitmix64(11, n_blocks)).astype(np.int32)
    table, dst = (np.full((len(lens), max(need)), -1, np.int32) for _ in range(2))
    at = 0
    for t in (table, dst):
        for s, nb in enumerate(need):
            t[s, :nb] = order[at:at + nb]
            at += nb
    rng = np.random.default_rng(2)
    keeps = [np.arange(33), np.sort(rng.permutation(200)[:90]), np.arange(0), np.array([74]), np.arange(0, 131, 3),
             np.arange(63, -1, -1), np.array([7, 7, 49, 0, 7, 21])]
    keep = np.zeros((len(lens), max(len(k) for k in keeps) + 2), np.int32)
    for s, k in enumerate(keeps):
        keep[s, :len(k)] = k
    codes, meta = (x.clone() for x in pool.read_codes())
    pool.compact(i32(table), i32(keep), i32([len(k) for k in keeps]), i32(dst))
    torch.cuda.synchronize()
    for s, k in enumerate(keeps):
        if len(k):
            a, b = slots(table[s], k), slots(dst[s], np.arange(len(k)))
            codes[torch.from_numpy(b)] = codes[torch.from_numpy(a)]
            meta[torch.from_numpy(b)] = meta[torch.from_numpy(a)]
    got_codes, got_meta = pool.read_codes()
    torch.cuda.synchronize()
    assert torch.equal(got_codes, codes) and torch.equal(got_meta, meta)


@pytest.mark.parametrize("mode,D,bits,Hkv", [MODES[0], MODES[5], MODES[7], MODES[12]])
def test_compact_leaves_out_what_is_not_there(gpu, mode, D, bits, Hkv):
    """Positions and pages out of range, counts past the list, destination rows
    with holes: those slots stay as they were, and nothing else is written."""
    import torch

    pool = filled(gpu, mode, D, bits, Hkv, 12)
    table = np.array([[0, 1, 2, 12], [3, -5, 2 ** 31 - 1, 4]], np.int32)
    dst = np.array([[6, 7], [8, -1]], np.int32)
    keep = np.array([[5, 64, -1, 33, 50, 2 ** 31 - 1, -2 ** 31, 18] + [17] * 12,
                     [0, 20, 40, 55, 3, 3, 3, 3] + [1] * 12], np.int32)
    codes, meta = (x.clone() for x in pool.read_codes())
    pool.compact(i32(table), i32(keep), i32([1000, 20]), i32(dst))
    torch.cuda.synchronize()
    for s in range(2):
        for i, p in enumerate(keep[s]):
            p = int(p)
            if not 0 <= p < 64 or not 0 <= table[s, p // 16] < 12 or dst[s, i // 16] < 0:
                continue
            a, b = table[s, p // 16] * 16 + p % 16, dst[s, i // 16] * 16 + i % 16
            codes[b], meta[b] = codes[a], meta[a]
    got_codes, got_meta = pool.read_codes()
    torch.cuda.synchronize()
    assert torch.equal(got_codes, codes) and torch.equal(got_meta, meta)


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", [(AFFINE, 256, 4, 8, 16), (AFFINE, 512, 8, 2, 16),
                                                (CODEBOOK, 256, 3, 2, 4), (PLAIN, 128, 16, 2, 4)])
def test_fork_slide_compact_and_attend(gpu, ora, mode, D, bits, Hkv, Hq):
    """A server's run: a prompt, a fork (shared pages, the last one copied in both
    layers), both branches decoding through a window with pages given back, then
    one compacted to its window and attended in full."""
    import torch

    window, sinks, n0, steps = 60, 5, 93, 40
    layers = [gpu.PagedPool(gpu.make_desc(Hkv, D, bits, mode=mode), 40) for _ in range(2)]
    book = gpu.PageBook(40)
    width = -(-(n0 + steps) // 16)
    a = book.alloc(-(-n0 // 16))
    k, v = (fast_kv(s, n0, Hkv, D, outliers=False) for s in (1, 2))
    zero = i32([0])
    for pool in layers:
        pool.append(dev_bf16(k[None]), dev_bf16(v[None]), i32([a]), zero)
    b, copy = book.fork(a, n0)
    assert copy is not None
    gpu.copy_blocks(layers, i32([copy[0]]), i32([copy[1]]))
    seqs, oracles = [a, b], []
    for _ in range(2):
        oc = ora.OracleCache(Hkv, D, bits, 0, n0 + steps + 1, mode=mode)
        oc.append(k, v)
        oracles.append(oc)
    for i in range(steps):
        n = n0 + i
        for s in range(2):
            seqs[s] = book.slide(seqs[s], n, window, sinks)
            if n % 16 == 0:
                seqs[s] = seqs[s] + book.alloc(1)
        table = i32([x + [-1] * (width - len(x)) for x in seqs])
        kn, vn = (np.stack([fast_kv(1000 + 4 * i + 2 * s + x, 1, Hkv, D, outliers=False) for s in range(2)])
                  for x in range(2))
        q = queries(77 + i, 2, Hq, Hkv, D)
        for s in range(2):
            oracles[s].append(kn[s], vn[s])
        outs = [pool.window_decode_step(dev_bf16(kn), dev_bf16(vn), table, i32([n, n]), i32([n + 1, n + 1]), n + 1,
                                        dev_bf16(q), window, sinks, D ** -0.5, dtype=torch.float32)
                for pool in layers]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        for s in range(2):
            check_window(outs[0][s], window_reference(ora, oracles[s], q[s], n, window, sinks, D ** -0.5), 6.0,
                         f"step {i} branch {s}")
    n = n0 + steps
    assert book.free_count() > 40 - 2 * (-(-window // 16) + 3)
    keep = np.array([j for j in range(n) if j < sinks or j > n - 1 - window], np.int32)
    fresh = book.alloc(-(-len(keep) // 16))
    table = i32([seqs[1] + [-1] * (width - len(seqs[1]))])
    layers[0].compact(table, i32([keep]), i32([len(keep)]), i32([fresh]))
    got = layers[0].attention(dev_bf16(q[1:]), i32([fresh]), i32([len(keep)]), len(keep), D ** -0.5,
                              dtype=torch.float32)
    torch.cuda.synchronize()
    check_window(got, outs[0][1:].double().cpu().numpy(), 12.0, "compacted")
    book.release(seqs[0])
    book.release(seqs[1])
    book.release(fresh)
    assert book.free_count() == 40


def test_page_calls_refuse(gpu):
    import torch

    lib, bad = gpu.load_library(), gpu.FMKV_ERR_INVALID_ARG
    pool = filled(gpu, *MODES[0], 8)
    before = pool.storage().clone()
    t, n = i32([[0, 1]]), i32([2])
    args = dict(tables=t.data_ptr(), width=2, keep=t.data_ptr(), most=2, n=n.data_ptr(), dst=t.data_ptr(), dwidth=2,
                seqs=1)
    for change in (dict(tables=None), dict(keep=None), dict(n=None), dict(dst=None), dict(width=0), dict(most=-1),
                   dict(dwidth=0), dict(seqs=-1), dict(seqs=65536), dict(most=33)):
        a = {**args, **change}
        assert lib.fmkv_paged_compact(pool._h, a["tables"], a["width"], a["keep"], a["most"], a["n"], a["dst"],
                                      a["dwidth"], a["seqs"], None) == bad, change
    for call in (lambda: gpu.copy_blocks([pool], t, t), lambda: gpu.copy_blocks([pool], n, i32([0, 1])),
                 lambda: gpu.copy_blocks([pool], n.long(), n), lambda: pool.compact(t, t, i32([1, 2]), t),
                 lambda: pool.compact(t, t.long(), n, t), lambda: pool.compact(t, t[0], n, t)):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()
    assert torch.equal(pool.storage(), before)


def test_storage_keeps_the_pool(gpu):
    """The storage tensor holds its pool: it outlives the pool's last name."""
    import gc

    import torch

    st = filled(gpu, *MODES[0], 3, seed=8).storage()
    gc.collect()
    want = torch.randint(0, 256, st.shape, generator=torch.Generator().manual_seed(8), dtype=torch.uint8)
    assert torch.equal(st.cpu(), want)
