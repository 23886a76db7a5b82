"""Accumulated attention weights of several queries per sequence, against
64-bit references; and the whole of an eviction by them."""
import numpy as np
import pytest

from gpu_util import dev_bf16, fast_kv
from shared_util import attend_reference, check_weights, poison_from
from window_util import AFFINE, CODEBOOK, PLAIN, TOKENS, Paged, check_window, queries

pytestmark = pytest.mark.gpu

# mode, bits, D, Hkv, Hq
FORMS = [(AFFINE, 4, 256, 8, 16), (AFFINE, 8, 512, 2, 16), (PLAIN, 16, 128, 4, 8), (AFFINE, 4, 128, 2, 2),
         (AFFINE, 8, 256, 1, 5), (AFFINE, 4, 512, 1, 8), (AFFINE, 8, 128, 3, 9), (CODEBOOK, 2, 128, 2, 4),
         (CODEBOOK, 3, 256, 2, 12), (CODEBOOK, 4, 512, 1, 7), (CODEBOOK, 2, 512, 2, 2), (PLAIN, 16, 512, 1, 8),
         (PLAIN, 16, 256, 2, 6), (CODEBOOK, 4, 256, 1, 1), (CODEBOOK, 3, 128, 2, 16), (CODEBOOK, 3, 512, 1, 3),
         (CODEBOOK, 2, 256, 1, 2), (CODEBOOK, 4, 128, 1, 4)]
# lengths after the queries, queries
BATCHES = [([1], 1), ([16, 17, 3, 33], 3), ([1000, 37, 333, 70], 37), ([2100], 130), ([5, 129, 0], 9)]


def reference(ora, oc, q, end, scale):
    """Sums over the queries q [n, Hq, D], the last at position end - 1."""
    total, n = np.zeros(max(end, 0)), len(q)
    for i in range(n):
        seen = end - n + i + 1
        if seen > 0:
            total[:seen] += attend_reference(ora, oc, q[i], seen, scale)[1]
    return total


@pytest.mark.parametrize("lens,n", BATCHES, ids=str)
@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", FORMS)
def test_attention_weights(gpu, ora, mode, bits, D, Hkv, Hq, lens, n):
    """Padded rows too: a sequence shorter than the queries begins below position 0."""
    import torch

    b = Paged(gpu, ora, mode, D, bits, Hkv, lens, seed=2)
    longest = max(lens)
    q = np.stack([queries(50 + s, n, Hq, Hkv, D) for s in range(len(lens))])
    want = [reference(ora, oc, q[s], t, D ** -0.5) for s, (oc, t) in enumerate(zip(b.oracles, lens))]
    start = b.lens_dev([t - n for t in lens])
    width = longest + 3
    old = (torch.rand((len(lens), width), generator=torch.Generator().manual_seed(3)) * 2).cuda()
    sums = torch.full((len(lens), width), 7.0, device="cuda")
    got = b.pool.attention_weights(dev_bf16(q), b.table(), start, longest, old, weights_out=sums, scale=D ** -0.5)
    assert got is sums
    for s, t in enumerate(lens):
        check_weights(sums[s, :t].double().cpu().numpy(), old[s, :t].double().cpu().numpy(), want[s], f"sequence {s}")
        assert (sums[s, t:] == 7.0).all()
    fresh = b.pool.attention_weights(dev_bf16(q), b.table(), start, longest, scale=D ** -0.5)
    for s, t in enumerate(lens):
        check_weights(fresh[s, :t].double().cpu().numpy(), np.zeros(t), want[s], f"from nothing {s}")
        assert not fresh[s, t:].any()
    again = old.clone()
    b.pool.attention_weights(dev_bf16(q), b.table(), start, longest, again, scale=D ** -0.5)
    for s, t in enumerate(lens):
        assert torch.equal(again[s, :t], sums[s, :t]) and torch.equal(again[s, t:], old[s, t:])


@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", [FORMS[0], FORMS[1], FORMS[2], FORMS[8]])
def test_many_rows_many_keys(gpu, ora, mode, bits, D, Hkv, Hq):
    """Enough tiles and keys that a work-group takes several of both: the sums of all
    queries of a prompt, the first ones' among them."""
    import torch

    T, n = 3000, 700
    b = Paged(gpu, ora, mode, D, bits, Hkv, [T, 1500], seed=4)
    q = np.stack([queries(70 + s, n, Hq, Hkv, D) for s in range(2)])
    sums = b.pool.attention_weights(dev_bf16(q), b.table(), b.lens_dev([T - n, 0]), T, scale=D ** -0.5)
    for s, (p0, end) in enumerate(((T - n, T), (0, n))):
        # in 64 bits, from the rows as the oracle holds them
        k = torch.from_numpy(b.oracles[s].dequant_kv(np.arange(end))[0]).cuda().double()
        qd = dev_bf16(q[s]).double()
        total = torch.zeros(end, dtype=torch.float64, device="cuda")
        hidden = torch.arange(end, device="cuda")[None] > torch.arange(p0, p0 + n, device="cuda")[:, None]
        for h in range(Hq):
            score = qd[:, h] @ k[:, h * Hkv // Hq].T.contiguous() * D ** -0.5
            total += torch.softmax(score.masked_fill(hidden, -torch.inf), -1).sum(0)
        check_weights(sums[s, :end].double().cpu().numpy(), np.zeros(end), total.cpu().numpy(), f"sequence {s}")
        assert not sums[s, end:].any()
        assert abs(float(sums[s].sum()) - n * Hq) < 1e-4 * n * Hq


@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", [FORMS[0], FORMS[1], FORMS[2], FORMS[8]])
def test_hidden_keys(gpu, ora, mode, bits, D, Hkv, Hq):
    """What the slots behind a sequence hold does not reach its sums."""
    import torch

    b = Paged(gpu, ora, mode, D, bits, Hkv, [200], seed=5)
    q = dev_bf16(queries(33, 5, Hq, Hkv, D)[None])
    start = b.lens_dev([60])
    want = b.pool.attention_weights(q, b.table(), start, 65, scale=D ** -0.5)
    poison_from(b, 0, 65)
    got = b.pool.attention_weights(q, b.table(), start, 65, scale=D ** -0.5)
    assert torch.equal(got, want) and bool(torch.isfinite(got).all())


@pytest.mark.parametrize("lens,n", [([300, 40], 2), ([400, 131], 45)], ids=str)
@pytest.mark.parametrize("power", [7, 12, 16])
@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", [f for f in FORMS if f[0] == AFFINE] + [(AFFINE, 8, 512, 1, 7), FORMS[2], FORMS[8]])
def test_large_queries(gpu, ora, mode, bits, D, Hkv, Hq, power, lens, n):
    """Queries whose sums over 64 dims and offset parts f16 does not hold, beside ordinary
    ones, over keys so much smaller: scores as everywhere else."""
    import torch

    b = Paged(gpu, ora, mode, D, bits, Hkv, lens, seed=2)
    for s, t in enumerate(lens):  # the same keys, times 2^-power (exact: bits of bf16)
        k, v = (fast_kv(10 * s + 2 + 5 * i, t, Hkv, D, outliers=False) for i in (0, 1))
        k = np.where(k & 0x7f80, k - (power << 7), 0).astype(np.uint16)
        b.oracles[s] = ora.OracleCache(Hkv, D, bits, 0, t + 1, mode=mode)
        b.oracles[s].append(k, v)
        b.pool.append(dev_bf16(k[None]), dev_bf16(v[None]), b.table(s),
                      torch.zeros(1, dtype=torch.int32, device="cuda"))
    q = np.stack([queries(50 + s, n, Hq, Hkv, D) for s in range(len(lens))])
    large = np.arange(n) % 3 != 1
    q[:, large] = np.where(q[:, large] & 0x7f80, q[:, large] + (power << 7), 0).astype(np.uint16)
    want = [reference(ora, oc, q[s], t, D ** -0.5) for s, (oc, t) in enumerate(zip(b.oracles, lens))]
    got = b.pool.attention_weights(dev_bf16(q), b.table(), b.lens_dev([t - n for t in lens]), max(lens),
                                   scale=D ** -0.5)
    for s, t in enumerate(lens):
        check_weights(got[s, :t].double().cpu().numpy(), np.zeros(t), want[s], f"sequence {s}")


@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", [FORMS[0], FORMS[2], FORMS[8]])
def test_no_queries(gpu, ora, mode, bits, D, Hkv, Hq):
    """An empty chunk adds nothing: what was accumulated, or zeros, of the positions
    before it, in a buffer that holds something else, and in place."""
    import torch

    lens = [300, 17, 0, 9]
    b = Paged(gpu, ora, mode, D, bits, Hkv, lens, seed=3)
    q = torch.empty((4, 0, Hq, D), dtype=torch.bfloat16, device="cuda")
    start = b.lens_dev([300, 17, 0, -2])
    seen = [300, 17, 0, 0]
    old = torch.rand((4, 303), generator=torch.Generator().manual_seed(1)).cuda()
    sums = torch.full((4, 303), 7.0, device="cuda")
    assert b.pool.attention_weights(q, b.table(), start, 300, old, weights_out=sums) is sums
    for s, t in enumerate(seen):
        assert torch.equal(sums[s, :t], old[s, :t]) and bool((sums[s, t:] == 7.0).all())
    sums.fill_(7.0)
    b.pool.attention_weights(q, b.table(), start, 300, weights_out=sums)
    for s, t in enumerate(seen):
        assert not sums[s, :t].any() and bool((sums[s, t:] == 7.0).all())
    same = old.clone()
    assert b.pool.attention_weights(q, b.table(), start, 300, same) is same
    assert torch.equal(same, old)


def test_graph(gpu, ora):
    import torch

    D, Hkv, Hq = 512, 2, 16
    b = Paged(gpu, ora, AFFINE, D, 8, Hkv, [900, 120], seed=8)
    q = dev_bf16(np.stack([queries(41 + s, 7, Hq, Hkv, D) for s in range(2)]))
    start, table = b.lens_dev([893, 113]), b.table()
    once = b.pool.attention_weights(q, table, start, 900, scale=D ** -0.5)
    acc = torch.zeros_like(once)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.pool.attention_weights(q, table, start, 900, acc, scale=D ** -0.5)
    total = torch.zeros_like(once)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        total = total + once
        assert torch.equal(acc, total)
        assert torch.equal(b.pool.attention_weights(q, table, start, 900, scale=D ** -0.5), once)


def test_eviction(gpu, ora):
    """A prompt's last queries weigh its positions, the heaviest stay, their tokens
    and weights move together, steps go on over what is left and weigh it, and it is cut again."""
    import torch

    D, bits, Hkv, Hq, mode = 256, 8, 2, 8, AFFINE
    lens, n, most, sinks, recent = [330, 41, 200], 16, 64, 4, 20
    b = Paged(gpu, ora, mode, D, bits, Hkv, lens, seed=12)
    scale = D ** -0.5
    q = np.stack([queries(60 + s, n, Hq, Hkv, D) for s in range(3)])
    sums = b.pool.attention_weights(dev_bf16(q), b.table(), b.lens_dev([t - n for t in lens]), max(lens), scale=scale)
    book = gpu.PageBook(64)
    pool = gpu.PagedPool(gpu.make_desc(Hkv, D, bits, mode=mode), b.n_blocks + 64)
    # both halves of the eviction in one pool: the prompt's blocks, then fresh ones
    pool.storage()[:b.n_blocks].copy_(b.pool.storage())
    room = most + 24
    fresh = torch.tensor([[b.n_blocks + x for x in book.alloc(-(-room // TOKENS))] for _ in lens],
                         dtype=torch.int32, device="cuda")
    acc = torch.full((3, room), 9.0, device="cuda")
    keep, n_keep, _ = gpu.heaviest_tokens(sums, b.lens_dev(), most, sinks, recent, weights_out=acc)
    pool.compact(b.table(), keep, n_keep, fresh)
    now = [min(t, most) for t in lens]
    assert n_keep.tolist() == now
    rows = [[oc.dequant_kv(np.array(keep[s, :t].tolist()))[i] for i in (0, 1)]
            for s, (oc, t) in enumerate(zip(b.oracles, now))]
    for s, t in enumerate(now):
        ids = keep[s, :t].tolist()
        assert ids == sorted(set(ids)) and ids[:sinks] == list(range(sinks))
        assert torch.equal(acc[s, :t], sums[s, ids]) and not acc[s, t:].any()
    total = acc.double().cpu().numpy()
    for step in range(20):
        kn, vn = (fast_kv(300 + 2 * step + i, 3, Hkv, D, outliers=False) for i in (0, 1))
        qs = queries(400 + step, 3, Hq, Hkv, D)
        for s in range(3):
            oc = ora.OracleCache(Hkv, D, bits, 0, 2, mode=mode)
            oc.append(kn[s:s + 1], vn[s:s + 1])
            rows[s] = [np.concatenate([r, x]) for r, x in zip(rows[s], oc.dequant_kv(np.array([0])))]
        now = [t + 1 for t in now]
        out, _ = pool.weighing_decode_step(
            dev_bf16(kn[:, None]), dev_bf16(vn[:, None]), fresh, b.lens_dev([t - 1 for t in now]), b.lens_dev(now),
            room, dev_bf16(qs), acc, scale=scale, dtype=torch.float32)

        class Rows:
            def __init__(self, kv):
                self.kv = kv

            def dequant_kv(self, at):
                return self.kv[0][at], self.kv[1][at]

        want = [attend_reference(ora, Rows(rows[s]), qs[s], now[s], scale) for s in range(3)]
        check_window(out, np.stack([w[0] for w in want]), 6.0, f"step {step}")
        for s in range(3):
            check_weights(acc[s, :now[s]].double().cpu().numpy(), total[s, :now[s]], want[s][1], f"step {step}")
            total[s] = acc[s].double().cpu().numpy()
    keep2, n2, kept2 = gpu.heaviest_tokens(acc, b.lens_dev(now), 32, sinks, 8)
    assert n2.tolist() == [32] * 3
    order = acc.cpu().numpy()
    for s, t in enumerate(now):
        mid = np.lexsort((np.arange(sinks, t - 8), -order[s, sinks:t - 8]))[:20] + sinks
        assert keep2[s].tolist() == sorted([*range(sinks), *mid.tolist(), *range(t - 8, t)])
        assert torch.equal(kept2[s], acc[s, keep2[s].long()])
