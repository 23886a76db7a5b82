"""Padded rows of a batched prefill: queries at positions below 0 get zeros, their keys
and values are stored nowhere, and every other sequence's results and slots are its own.
(Lengths of 0 are starts of -n; the table entries before a sequence's first are another's.)"""
import numpy as np
import pytest
import torch

from gpu_util import dev_bf16, fast_kv
from window_util import AFFINE, CODEBOOK, PLAIN, Paged, check_window, queries, window_reference

pytestmark = pytest.mark.gpu

CONFIGS = [  # mode, D, bits, Hkv, Hq
    (AFFINE, 256, 4, 8, 16), (AFFINE, 512, 8, 2, 16), (AFFINE, 128, 4, 1, 3), (CODEBOOK, 256, 3, 2, 4),
    (PLAIN, 128, 16, 2, 4),
]
N = 21
# before the padding ends, at it, a part of the row past it, ordinary ones between
STARTS = [60, -N, 33, -16, -1, -20, -1000, 0, -2 ** 31, -N - 1]


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", CONFIGS)
@pytest.mark.parametrize("window", [10, 4000])
@pytest.mark.parametrize("hole", [-1, 0])
def test_padded_prefill_steps(gpu, ora, mode, D, bits, Hkv, Hq, window, hole):
    """The windowed step and the plain one over the same rows. Table entries of what
    does not exist are -1 or another sequence's block."""
    lens = [max(x, 0) for x in STARTS]
    p = Paged(gpu, ora, mode, D, bits, Hkv, lens, room=N, dirty=False)
    for s, x in enumerate(STARTS):
        p.tables[s, max(-(-(x + N) // 16), 0):] = hole  # (block 0 is some sequence's)
    k, v = (np.stack([fast_kv(90 + s + y, N, Hkv, D, outliers=False) for s in range(len(STARTS))]) for y in (0, 40))
    q = np.stack([queries(7 + s, N, Hq, Hkv, D) for s in range(len(STARTS))])
    before = p.pool.storage().clone()
    for s, x in enumerate(STARTS):
        if x + N > 0:
            p.oracles[s].append(k[s, max(-x, 0):], v[s, max(-x, 0):])
    args = (dev_bf16(k), dev_bf16(v), p.table(), p.lens_dev(STARTS), dev_bf16(q))
    written = {int(p.tables[s, j // 16]) for s, x in enumerate(STARTS) for j in range(max(x, 0), max(x + N, 0))}
    rest = torch.tensor([b not in written for b in range(p.n_blocks)])
    for plain in (False, True):
        if plain:
            out = p.pool.prefill_step(*args, D ** -0.5, dtype=torch.float32)
        else:
            out = p.pool.window_prefill_step(*args, window, 3, D ** -0.5, dtype=torch.float32)
        torch.cuda.synchronize()
        for s, x in enumerate(STARTS):
            for i in range(N):
                ref = window_reference(ora, p.oracles[s], q[s, i], x + i, 1 << 30 if plain else window, 3, D ** -0.5)
                check_window(out[s, i], ref, 6.0, f"plain {plain} start {x} row {i}")
        st = p.pool.storage()
        assert torch.equal(st[rest], before[rest])
        codes, meta = p.pool.read_codes()
        torch.cuda.synchronize()
        for s, x in enumerate(STARTS):
            pos = np.arange(max(x + N, 0))
            at = p.tables[s, pos // 16].astype(np.int64) * 16 + pos % 16
            assert np.array_equal(codes[torch.from_numpy(at).cuda()].cpu().numpy().view(np.uint32),
                                  p.oracles[s].codes[:len(pos)]), f"start {x}"
    again = p.pool.window_prefill(*args[4:], *args[2:4], window, 3, D ** -0.5, dtype=torch.float32)
    p.pool.append(*args[:4])
    once = p.pool.storage().clone()
    torch.cuda.synchronize()
    assert torch.equal(once, p.pool.storage())
    for s, x in enumerate(STARTS):
        assert not bool(again[s, :min(max(-x, 0), N)].any()), f"start {x}"
