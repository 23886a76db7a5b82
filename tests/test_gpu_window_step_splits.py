"""The windowed decode step where a split holds eight blocks and more: the affine
kernel's single-wave streams (packed columns and not) with the new token's column,
whose slot they leave out; the other modes at the same plans. Before each step the
slots that it does not see hold NaNs and infinities, the new token's among them, and
pages without visible slots are given back."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from gpu_util import check_codes, dev_bf16, fast_kv
from window_util import AFFINE, CODEBOOK, PLAIN, Paged, check_window, queries, window_reference

pytestmark = pytest.mark.gpu

CONFIGS = [  # mode, D, bits, Hkv, Hq
    (AFFINE, 256, 4, 8, 16), (AFFINE, 256, 4, 2, 12), (AFFINE, 128, 4, 1, 3), (AFFINE, 128, 8, 4, 8),
    (AFFINE, 512, 8, 2, 16), (CODEBOOK, 256, 3, 2, 4), (PLAIN, 256, 16, 2, 4),
]
# empty, inside the window, about its size, past it with a gap to the sinks; block ends
LENS = [0, 5, 127, 128, 299, 301, 340, 615, 1000]


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq", CONFIGS)
@pytest.mark.parametrize("bps", [8, 9, 64])
@pytest.mark.parametrize("window,sinks", [(301, 43), (1, 17)])
def test_window_decode_step_of_long_splits(gpu, ora, mode, D, bits, Hkv, Hq, bps, window, sinks):
    p = Paged(gpu, ora, mode, D, bits, Hkv, LENS, room=3)
    pages = p.tables.copy()
    gpu.set_blocks_per_split(bps)
    try:
        for step in range(3):
            now = [n + step for n in LENS]
            p.hide(now, now, window, sinks)
            for s, n in enumerate(now):  # (pages of later steps are not given back)
                p.tables[s, n // 16 + 1:] = pages[s, n // 16 + 1:]
            k, v = (np.stack([fast_kv(500 + 50 * step + s + x, 1, Hkv, D, outliers=False)
                              for s in range(len(LENS))]) for x in (0, 25))
            q = np.stack([queries(300 + 10 * step + s, 1, Hq, Hkv, D)[0] for s in range(len(LENS))])
            out = p.pool.window_decode_step(dev_bf16(k), dev_bf16(v), p.table(), p.lens_dev(now),
                                            p.lens_dev([n + 1 for n in now]), max(now) + 1, dev_bf16(q), window,
                                            sinks, D ** -0.5, dtype=torch.float32)
            codes, meta = p.pool.read_codes()
            torch.cuda.synchronize()
            for s, n in enumerate(now):
                p.oracles[s].append(k[s], v[s])
                ref = window_reference(ora, p.oracles[s], q[s], n, window, sinks, D ** -0.5)
                check_window(out[s], ref, 6.0, f"step {step} position {n}")
                slot = int(pages[s, n // 16]) * 16 + n % 16
                stored = SimpleNamespace(codes=p.oracles[s].codes[n:n + 1], meta=p.oracles[s].meta[n:n + 1])
                check_codes(codes[slot:slot + 1], meta[slot:slot + 1], stored, what=f"step {step} sequence {s}")
    finally:
        gpu.set_blocks_per_split(0)
