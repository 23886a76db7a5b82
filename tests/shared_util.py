"""Batches whose sequences share prefixes, and references of accumulated
attention weights in 64 bits, for the tests of both."""
import numpy as np

import synth
from gpu_util import dev_bf16, fast_kv
from window_util import TOKENS, poison


class Shared:
    """Sequences in groups: groups[g] = (prefix, [lengths]); `alone`: lengths of the
    sequences before the first group and after the last one. A member's table begins with
    the blocks of its group's first one, the prefix's whole blocks; what it holds
    behind them is its own. Unwritten slots are full of NaNs; other entries of the tables
    name no block."""

    def __init__(self, gpu, ora, mode, D, bits, Hkv, groups, alone=((), ()), seed=1, room=0):
        import torch

        self.gpu, self.mode, self.D, self.bits, self.Hkv = gpu, mode, D, bits, Hkv
        rows = [(0, n, None) for n in alone[0]]
        self.starts = [len(rows)]
        for g, (prefix, lens) in enumerate(groups):
            rows += [(prefix, n, g) for n in lens]
            self.starts.append(len(rows))
        rows += [(0, n, None) for n in alone[1]]
        self.prefix, self.lens = [r[0] for r in rows], [r[1] for r in rows]
        self.rest = [n - min(p, n) // TOKENS * TOKENS if g is not None else n for p, n, g in rows]
        self.width = max(1, max((n + room + TOKENS - 1) // TOKENS for n in self.lens))
        n_blocks = sum((n + room + TOKENS - 1) // TOKENS for n in self.lens) + 3
        order = iter(np.argsort(synth.splitmix64(177 + seed, n_blocks)).astype(np.int32))
        self.pool = gpu.PagedPool(gpu.make_desc(Hkv, D, bits, mode=mode), n_blocks)
        self.pool.storage().fill_(0xff)
        self.tables = np.full((len(rows), self.width), -1, np.int32)
        self.oracles, first, head = [], {}, {}
        for s, (prefix, n, g) in enumerate(rows):
            shared = 0
            if g is not None and prefix:
                if g not in head:
                    head[g] = [fast_kv(900 * g + seed + i, prefix, Hkv, D, outliers=False) for i in (0, 7)]
                    first[g] = s
                else:
                    shared = min(min(prefix, n) // TOKENS, min(prefix, self.lens[first[g]]) // TOKENS)
            self.tables[s, :shared] = self.tables[first[g], :shared] if shared else 0
            for b in range(shared, (n + room + TOKENS - 1) // TOKENS):
                self.tables[s, b] = next(order)
            own = [fast_kv(10 * s + seed + i, max(n, 1), Hkv, D, outliers=False) for i in (3, 5)]
            if g is not None and prefix:
                m = min(prefix, n)
                for i in range(2):
                    own[i][:m] = head[g][i][:m]
            oc = ora.OracleCache(Hkv, D, bits, 0, n + room + 1, mode=mode)
            if n:
                oc.append(own[0][:n], own[1][:n])
                at = shared * TOKENS
                if n > at:
                    self.pool.append(dev_bf16(own[0][None, at:n]), dev_bf16(own[1][None, at:n]),
                                     self.table([s]), torch.tensor([at], dtype=torch.int32, device="cuda"))
            self.oracles.append(oc)
        torch.cuda.synchronize()

    def table(self, rows=None):
        import torch

        t = self.tables if rows is None else self.tables[rows]
        return torch.from_numpy(np.ascontiguousarray(t)).cuda()

    def ints(self, x):
        import torch

        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def args(self):
        """block_tables, seq_lens, prefix_lens, group_starts, the bounds."""
        return (self.table(), self.ints(self.lens), self.ints(self.prefix), self.ints(self.starts),
                max(self.prefix), max(max(self.rest), 1))


def poison_from(paged, s, first):
    """Every slot of sequence s from position `first` on made not a number."""
    st = paged.pool.storage()
    for j in range(first, paged.width * TOKENS):
        b = int(paged.tables[s, j // TOKENS])
        if b >= 0:
            poison(st, b, j % TOKENS, paged.D, paged.bits, paged.mode)


def attend_reference(ora, oc, q, n, scale):
    """f64 attention of q [Hq, D] over the oracle's first n rows, and the weights
    summed over the heads."""
    if n < 1:
        return np.zeros(q.shape), np.zeros(0)
    k, v = oc.dequant_kv(np.arange(n))
    qf = ora.bf16_to_f32(q).astype(np.float64)
    group = qf.shape[0] // k.shape[1]
    out, total = np.empty(qf.shape), np.zeros(n)
    for h in range(qf.shape[0]):
        s = (k[:, h // group].astype(np.float64) @ qf[h]) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        total += p
        out[h] = p @ v[:, h // group].astype(np.float64)
    return out, total


def check_weights(out, before, new, what=""):
    """Scores of soft scales stay below 64 in base 2 and come out of at most 32
    roundings each: off by 64 * 32 * 2^-24 = 2^-13 at most, so a weight, by itself
    and through its sum, by 2 ln 2 times that, and by a few roundings of its own:
    together below 2^-12 of it; the sum over the heads and with what was there by at most
    64 roundings of half a step, 2^-18 of it. Where nothing is added, nothing changes."""
    err = np.abs(out.astype(np.float64) - (before + new))
    allow = 2.0 ** -12 * new + 2.0 ** -18 * np.where(new > 0, new, 0) + 2.0 ** -24 * np.abs(before + new)
    bad = ~(err <= allow)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} weights off, first at {np.argwhere(bad)[0]}, "
                           f"{np.nanmax(err / (new + 1e-30)):.3e} of its own")
