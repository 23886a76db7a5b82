"""Padded rows of a batched decode step, with a window and without, of one token and of
three: rows of length 0 and below store nothing and get zeros, the others are theirs."""
import numpy as np
import pytest
import torch

from gpu_util import dev_bf16, fast_kv
from window_util import AFFINE, CODEBOOK, PLAIN, Paged, check_window, queries, window_reference

pytestmark = pytest.mark.gpu

CONFIGS = [  # mode, D, bits, Hkv, Hq
    (AFFINE, 256, 4, 8, 16), (AFFINE, 512, 8, 2, 16), (CODEBOOK, 256, 3, 2, 4), (PLAIN, 128, 16, 2, 4),
]
LENS = [70, 0, 33, -6, -2 ** 31, 1]  # after the step


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", CONFIGS)
@pytest.mark.parametrize("n,window", [(1, 20), (1, 0), (3, 0)])
@pytest.mark.parametrize("hole", [-1, 0])
def test_padded_decode_steps(gpu, ora, mode, D, bits, Hkv, Hq, n, window, hole):
    start = [max(x - n, -2 ** 31) for x in LENS]
    p = Paged(gpu, ora, mode, D, bits, Hkv, [max(x, 0) for x in start], room=n, dirty=False)
    for s, x in enumerate(LENS):
        p.tables[s, max(-(-x // 16), 0):] = hole  # (block 0 is some sequence's)
    k, v = (np.stack([fast_kv(9 + s + y, n, Hkv, D, outliers=False) for s in range(len(LENS))]) for y in (0, 40))
    q = np.stack([queries(7 + s, 1, Hq, Hkv, D)[0] for s in range(len(LENS))])
    before = p.pool.storage().clone()
    for s, x in enumerate(LENS):
        if x > 0:
            p.oracles[s].append(k[s, max(-start[s], 0):], v[s, max(-start[s], 0):])
    args = (dev_bf16(k), dev_bf16(v), p.table(), p.lens_dev(start), p.lens_dev(LENS), max(LENS), dev_bf16(q))
    if window:
        out = p.pool.window_decode_step(*args, window, 3, D ** -0.5, dtype=torch.float32)
    else:
        out = p.pool.decode_step(*args, D ** -0.5, dtype=torch.float32)
    torch.cuda.synchronize()
    for s, x in enumerate(LENS):
        ref = window_reference(ora, p.oracles[s], q[s], max(x, 0) - 1, window or 1 << 30, 3, D ** -0.5)
        check_window(out[s], ref, 6.0, f"length {x}")
    written = {int(p.tables[s, j // 16]) for s, x in enumerate(LENS) for j in range(max(x - n, 0), max(x, 0))}
    rest = torch.tensor([b not in written for b in range(p.n_blocks)])
    assert torch.equal(p.pool.storage()[rest], before[rest])
