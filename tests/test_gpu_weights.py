"""Accumulated attention weights and the positions that an eviction by them
keeps, against 64-bit references and a sort."""
import numpy as np
import pytest

from gpu_util import check_codes, dev_bf16, fast_kv
from shared_util import attend_reference, check_weights
from window_util import AFFINE, CODEBOOK, PLAIN, TOKENS, Paged, check_window, queries

pytestmark = pytest.mark.gpu

# mode, bits, D, Hkv, Hq
FORMS = [(AFFINE, 4, 256, 8, 16), (AFFINE, 8, 512, 2, 16), (PLAIN, 16, 128, 4, 8), (AFFINE, 4, 128, 2, 2),
         (AFFINE, 8, 256, 1, 5), (AFFINE, 4, 512, 1, 8), (AFFINE, 8, 128, 3, 9), (CODEBOOK, 2, 128, 2, 4),
         (CODEBOOK, 3, 256, 2, 12), (CODEBOOK, 4, 512, 1, 7), (CODEBOOK, 2, 512, 2, 2), (PLAIN, 16, 512, 1, 8),
         (PLAIN, 16, 256, 2, 6), (CODEBOOK, 4, 256, 1, 1), (CODEBOOK, 3, 128, 2, 16), (AFFINE, 4, 256, 17, 68)]
LENS = [[1], [16, 17, 1, 0, 15], [1000, 37, 333], [4097]]


def host(t):
    return t.double().cpu().numpy()


def before(n, width, seed):
    import torch

    g = torch.Generator().manual_seed(seed)
    return (torch.rand((n, width), generator=g) * 3).cuda()


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", FORMS)
def test_weighing_attention(gpu, ora, mode, bits, D, Hkv, Hq, lens):
    import torch

    b = Paged(gpu, ora, mode, D, bits, Hkv, lens, seed=2)
    n, longest = len(lens), max(lens)
    q = queries(21, n, Hq, Hkv, D)
    want = [attend_reference(ora, oc, q[s], t, D ** -0.5) for s, (oc, t) in enumerate(zip(b.oracles, lens))]
    vmax = max(float(np.abs(oc.dequant_kv(np.arange(t))[1]).max()) for oc, t in zip(b.oracles, lens) if t)
    width = longest + 5
    acc = before(n, width, 4)
    old = host(acc)
    sums = torch.full((n, width), 7.0, device="cuda")
    out, got = b.pool.weighing_attention(dev_bf16(q), b.table(), b.lens_dev(), longest, acc, weights_out=sums,
                                         scale=D ** -0.5, dtype=torch.float32)
    assert got is sums and np.array_equal(host(acc), old)
    check_window(out, np.stack([w[0] for w in want]), vmax, "output")
    for s, t in enumerate(lens):
        check_weights(host(sums)[s, :t], old[s, :t], want[s][1], f"sequence {s}")
    assert all((host(sums)[s, t:] == 7.0).all() for s, t in enumerate(lens))
    # in place, and from nothing
    same, got = b.pool.weighing_attention(dev_bf16(q), b.table(), b.lens_dev(), longest, acc, scale=D ** -0.5,
                                          dtype=torch.float32)
    assert got is acc and torch.equal(same, out)
    assert all(torch.equal(acc[s, :t], sums[s, :t]) and np.array_equal(host(acc)[s, t:], old[s, t:])
               for s, t in enumerate(lens))
    out16, fresh = b.pool.weighing_attention(dev_bf16(q), b.table(), b.lens_dev(), longest, scale=D ** -0.5)
    check_window(out16, np.stack([w[0] for w in want]), vmax, "bf16")
    for s, t in enumerate(lens):
        check_weights(host(fresh)[s, :t], np.zeros(t), want[s][1], f"from nothing {s}")
        assert not fresh[s, t:].any()


@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", FORMS)
def test_weighing_step(gpu, ora, mode, bits, D, Hkv, Hq):
    """Steps from an empty sequence on, across a block's end, with a padded row."""
    import torch

    lens = [0, 30, 15, 200]
    b = Paged(gpu, ora, mode, D, bits, Hkv, lens, seed=6, room=4)
    n, padded = len(lens), 2
    acc = torch.zeros((n, 210), device="cuda")
    total = np.zeros((n, 210))
    for step in range(3):
        k, v = (fast_kv(700 + 10 * step + i, n, Hkv, D, outliers=False) for i in (0, 1))
        q = queries(90 + step, n, Hq, Hkv, D)
        now = [t + step + 1 for t in lens]
        now[padded] = 0
        for s in range(n):
            if s != padded:
                b.oracles[s].append(k[s:s + 1], v[s:s + 1])
        want = [attend_reference(ora, oc, q[s], t, D ** -0.5) for s, (oc, t) in enumerate(zip(b.oracles, now))]
        old = host(acc)
        out, _ = b.pool.weighing_decode_step(
            dev_bf16(k[:, None]), dev_bf16(v[:, None]), b.table(), b.lens_dev([t - 1 for t in now]), b.lens_dev(now),
            max(now), dev_bf16(q), acc, scale=D ** -0.5, dtype=torch.float32)
        check_window(out, np.stack([w[0] for w in want]), 6.0, f"step {step}")
        for s, t in enumerate(now):
            check_weights(host(acc)[s, :t], old[s, :t], want[s][1], f"step {step}, sequence {s}")
            total[s, :t] += want[s][1]
            assert np.array_equal(host(acc)[s, t:], old[s, t:])
    codes, meta = b.pool.read_codes()
    for s in range(n):
        at = np.arange(lens[s] + 3 if s != padded else lens[s])
        slots = torch.from_numpy(b.tables[s, at // TOKENS] * TOKENS + at % TOKENS).long().cuda()
        check_codes(codes[slots], meta[slots], b.oracles[s], slots=at, what=f"sequence {s}")


@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", [(CODEBOOK, 4, 128, 2, 6), (CODEBOOK, 2, 256, 1, 8), (CODEBOOK, 3, 512, 1, 4)])
def test_weighing_other_codebooks(gpu, ora, mode, bits, D, Hkv, Hq):
    """The widths that are not among the forms above, over slots full of NaNs."""
    for lens in LENS:
        test_weighing_attention(gpu, ora, mode, bits, D, Hkv, Hq, lens)
    test_weighing_step(gpu, ora, mode, bits, D, Hkv, Hq)


def test_weighing_graph(gpu, ora):
    """A captured call replayed with eager ones between: each replay adds the same."""
    import torch

    D, Hkv, Hq = 256, 8, 16
    b = Paged(gpu, ora, AFFINE, D, 4, Hkv, [500, 900, 20], seed=8)
    q, lens, table = dev_bf16(queries(31, 3, Hq, Hkv, D)), b.lens_dev(), b.table()
    want, once = b.pool.weighing_attention(q, table, lens, 900, scale=D ** -0.5)
    acc, out = torch.zeros_like(once), torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.pool.weighing_attention(q, table, lens, 900, acc, scale=D ** -0.5, out=out)
    total = torch.zeros_like(once)
    for _ in range(4):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        total = total + once
        assert torch.equal(out, want) and torch.equal(acc, total)
        again, sums = b.pool.weighing_attention(q, table, lens, 900, scale=D ** -0.5)
        assert torch.equal(again, want) and torch.equal(sums, once)


# ---------------------------------------------------------------------------
# the positions that are kept
# ---------------------------------------------------------------------------

def keep_reference(w, t, most, sinks, recent):
    t = min(max(t, 0), len(w))
    if t <= most:
        return np.arange(t)
    key = np.where(np.isnan(w), -np.inf, w)
    mid = np.arange(sinks, t - recent)
    # (a NaN after an infinitely light weight)
    order = np.lexsort((mid, np.isnan(w[mid]), -key[mid]))
    return np.sort(np.concatenate([np.arange(sinks), mid[order[:most - sinks - recent]], np.arange(t - recent, t)]))


def kept(gpu, w, lens, most, sinks, recent, room=3, **kw):
    import torch

    n = len(lens)
    wd = torch.from_numpy(w).cuda()
    keep = torch.full((n, most), -9, dtype=torch.int32, device="cuda")
    out = torch.full((n, most + room), 5.0, device="cuda")
    k, nk, o = gpu.heaviest_tokens(wd, torch.tensor(lens, dtype=torch.int32, device="cuda"), most, sinks, recent,
                                   keep=keep, weights_out=out, **kw)
    assert k is keep and o is out
    k, nk, o = (x.cpu().numpy() for x in (k, nk, o))
    for s, t in enumerate(lens):
        want = keep_reference(w[s], t, most, sinks, recent)
        assert nk[s] == len(want)
        assert np.array_equal(k[s, :nk[s]], want), f"sequence {s} of {t}"
        assert (k[s, nk[s]:] == -9).all()
        assert np.array_equal(o[s, :nk[s]], w[s][want], equal_nan=True)
        assert not o[s, nk[s]:].any()


def values(kind, n, width, seed):
    rng = np.random.default_rng(seed)
    if kind == "heavy":
        return np.exp(3 * rng.standard_normal((n, width))).astype(np.float32)
    if kind == "ties":
        return rng.integers(0, 5, (n, width)).astype(np.float32) / 8
    if kind == "zeros":  # of both signs, all equal
        return np.where(rng.random((n, width)) < 0.5, 0.0, -0.0).astype(np.float32)
    if kind == "signs":
        return rng.standard_normal((n, width)).astype(np.float32)
    w = rng.standard_normal((n, width)).astype(np.float32)  # "special"
    at = rng.random((n, width))
    w[at < 0.3] = np.nan
    w[(at > 0.3) & (at < 0.4)] = np.inf
    w[(at > 0.4) & (at < 0.5)] = -np.inf
    w[(at > 0.5) & (at < 0.55)] = np.float32(1e-42)
    w[(at > 0.55) & (at < 0.6)] = -np.nan
    return w


@pytest.mark.parametrize("kind", ["heavy", "ties", "zeros", "signs", "special"])
@pytest.mark.parametrize("width,lens,most,sinks,recent", [
    (1, [1, 0, -3], 1, 0, 0), (40, [40, 17, 16, 41, 200], 16, 4, 5), (100, [100, 99, 3], 7, 7, 0),
    (100, [100, 60], 60, 0, 60), (130, [130, 129], 128, 1, 2), (2000, [2000, 1025, 1024, 1500], 1024, 3, 100),
    (5003, [5003], 1, 0, 0), (40001, [40001, 33000, 70], 4097, 4, 1000), (70000, [70000, 65537], 66000, 0, 1),
    (300001, [300001], 2048, 4, 64)])
def test_kept_positions(gpu, kind, width, lens, most, sinks, recent):
    kept(gpu, values(kind, len(lens), width, 5), lens, most, sinks, recent)


def test_kept_of_many(gpu):
    rng = np.random.default_rng(3)
    lens = [int(x) for x in rng.integers(0, 3000, 300)]
    kept(gpu, values("ties", 300, 3000, 9), lens, 700, 2, 50, room=0)


def test_kept_without_weights_out_and_captured(gpu):
    import torch

    w = torch.from_numpy(values("heavy", 3, 900, 2)).cuda()
    lens = torch.tensor([900, 100, 650], dtype=torch.int32, device="cuda")
    want = gpu.heaviest_tokens(w, lens, 256, 4, 32)
    keep, n_keep, out = (torch.zeros_like(x) for x in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.heaviest_tokens(w, lens, 256, 4, 32, keep=keep, n_keep=n_keep, weights_out=out)
    for _ in range(3):
        keep.zero_(), n_keep.zero_(), out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((keep, n_keep, out), want))
        gpu.heaviest_tokens(w, lens, 300, 4, 32)
    lib = gpu.load_library()
    keep.zero_()
    assert lib.fmkv_heaviest_tokens(w.data_ptr(), 900, lens.data_ptr(), 3, 256, 4, 32, keep.data_ptr(),
                                    n_keep.data_ptr(), None, 0, None) == gpu.FMKV_OK
    torch.cuda.synchronize()
    assert torch.equal(keep, want[0])
