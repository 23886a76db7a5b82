"""Window prefill of a few more tiles than run at once: the last tiles' keys are split
into ranges. Tails over several sequences and KV heads, short sequences in them (ranges
without a key), long ones whose window lies past the sinks; hidden slots hold NaNs and
infinities and pages without visible slots are given back."""
import gc

import numpy as np
import pytest
import torch

from gpu_util import dev_bf16
from window_util import AFFINE, CODEBOOK, PLAIN, Paged, check_window, queries, window_reference

pytestmark = pytest.mark.gpu

WINDOW, SINKS = 1200, 100
# The most steps (two blocks) of a tile of 64 rows: its window, positions and sinks
STEPS = ((WINDOW + 64 + 14) // 16 + 1 + -(-SINKS // 16)) // 2 + 2

CASES = [  # mode, D, bits, Hkv, Hq, sequences, queries of each, work-groups that run at once on 256 CUs
    (AFFINE, 512, 8, 2, 16, 22, 56, 256), (CODEBOOK, 512, 4, 2, 16, 22, 56, 256),
    (AFFINE, 256, 4, 8, 16, 34, 40, 512), (PLAIN, 256, 16, 4, 8, 45, 90, 512),
    (CODEBOOK, 128, 3, 4, 4, 50, 200, 768), (AFFINE, 128, 8, 4, 4, 53, 260, 1024),
]
# starts of the last sequences: the long ones, none before, one, a gap between sinks and window
ENDS = [(2900, 0, 3, 1700), (1700, 2900, 1, 0)]


@pytest.mark.parametrize("mode,D,bits,Hkv,Hq,seqs,n,once", CASES)
@pytest.mark.parametrize("ends", ENDS)
def test_window_prefill_split_tail(gpu, ora, mode, D, bits, Hkv, Hq, seqs, n, once, ends):
    start = [(7 * s) % 40 for s in range(seqs - len(ends))] + list(ends)
    p = Paged(gpu, ora, mode, D, bits, Hkv, [x + n for x in start])
    # what the plan comes to on 256 CUs: a tail over several heads and sequences
    tile = 64 // (Hq // Hkv)
    total = -(-n // tile) * Hkv * seqs
    tail = total - once
    ranges = min((768 if D == 128 else once) // tail, STEPS // 8)
    assert 0 < tail < total // 4 and tail > -(-n // tile) * Hkv and ranges >= 3 and STEPS - STEPS // ranges >= 24
    p.hide(start, [x + n - 1 for x in start], WINDOW, SINKS)
    q = np.stack([queries(4 + s, n, Hq, Hkv, D) for s in range(seqs)])
    qd, table, first = dev_bf16(q), p.table(), p.lens_dev(start)

    def call(out):
        return p.pool.window_prefill(qd, table, first, WINDOW, SINKS, D ** -0.5, out=out)

    held, eager, again = (torch.zeros(qd.shape, dtype=torch.float32, device="cuda") for _ in range(3))
    gc.collect()  # (what earlier tests held, and a capture would give back)
    torch.cuda.empty_cache()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(held)
    torch.cuda.synchronize()
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        # (a captured call's partial rows are in the pool's workspace: it was split)
        assert before - torch.cuda.mem_get_info()[0] >= tail * ranges * 64 * (D + 2) * 4
    call(eager)
    torch.cuda.synchronize()
    for s in [0, seqs // 2, *range(seqs - 6, seqs)]:
        for i in (0, 1, n // 2, n - 1):
            ref = window_reference(ora, p.oracles[s], q[s, i], start[s] + i, WINDOW, SINKS, D ** -0.5)
            check_window(eager[s, i], ref, 6.0, f"sequence {s} row {i} position {start[s] + i}")
    for _ in range(3):
        held.fill_(7.0)
        graph.replay()
        call(again)
        torch.cuda.synchronize()
        assert torch.equal(held, eager) and torch.equal(again, eager)
