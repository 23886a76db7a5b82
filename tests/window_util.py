"""Paged pools for the tests of windowed attention and page operators: shuffled
pages, pages given back (-1), slots that hold anything, references in 64 bits."""
import numpy as np

import synth
from gpu_util import dev_bf16, fast_kv, fast_q

AFFINE, CODEBOOK, PLAIN = 0, 1, 2
TOKENS = 16


def layout(D, bits, mode):
    """(bytes of K or V codes, of K or V scale / bias or norms, of a head-block)."""
    code = TOKENS * D * bits // 8
    meta = {AFFINE: D, CODEBOOK: 2 * TOKENS, PLAIN: 0}[mode]
    step = (meta + 63) // 64 * 64
    return code, step, (2 * code + 2 * step + 255) // 256 * 256


def poison(storage, block, token, D, bits, mode):
    """Makes a slot of a pool's storage (uint8 [blocks, heads, bytes]) not a
    number: what scales its V (and, where stored as they are, V itself) and its K."""
    code, step, _ = layout(D, bits, mode)
    b = storage[block]
    if mode == AFFINE:
        for r in range(2):
            for g in range(D // 64):
                o = 2 * code + r * step + (g * TOKENS + token) * 4
                b[:, o:o + 4] = 0xff  # f16 NaN scale and bias
    elif mode == CODEBOOK:
        for r in range(2):
            o = 2 * code + r * step + 2 * token
            b[:, o], b[:, o + 1] = 0x00, 0x7c  # f16 infinity
    else:
        b[:, token * 2 * D:(token + 1) * 2 * D] = 0xff
        for d in range(D):
            o = code + d * 2 * TOKENS + 2 * token
            b[:, o], b[:, o + 1] = 0x80, 0x7f  # bf16 infinity


class Paged:
    """n sequences of `lens` tokens in a pool of shuffled pages, every unwritten
    slot full of NaNs (dirty), and the oracle of each."""

    def __init__(self, gpu, ora, mode, D, bits, Hkv, lens, seed=1, room=0, spare=3, dirty=True):
        import torch

        self.gpu, self.mode, self.D, self.bits, self.Hkv, self.lens = gpu, mode, D, bits, Hkv, list(lens)
        need = [(n + room + TOKENS - 1) // TOKENS for n in lens]
        self.width = max(1, max(need))
        self.n_blocks = sum(need) + spare
        order = np.argsort(synth.splitmix64(77 + seed, self.n_blocks)).astype(np.int32)
        self.tables = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for s, nb in enumerate(need):
            self.tables[s, :nb] = order[at:at + nb]
            at += nb
        self.spare = order[at:]
        self.pool = gpu.PagedPool(gpu.make_desc(Hkv, D, bits, mode=mode), self.n_blocks)
        if dirty:
            self.pool.storage().fill_(0xff)
        self.oracles = []
        for s, n in enumerate(lens):
            oc = ora.OracleCache(Hkv, D, bits, 0, n + room + 1, mode=mode)
            if n:
                k, v = fast_kv(10 * s + seed, n, Hkv, D, outliers=False), fast_kv(10 * s + seed + 5, n, Hkv, D, outliers=False)
                oc.append(k, v)
                self.pool.append(dev_bf16(k[None]), dev_bf16(v[None]), self.table(s),
                                 torch.zeros(1, dtype=torch.int32, device="cuda"))
            self.oracles.append(oc)
        torch.cuda.synchronize()

    def table(self, s=None):
        import torch

        t = self.tables if s is None else self.tables[s:s + 1]
        return torch.from_numpy(np.ascontiguousarray(t)).cuda()

    def lens_dev(self, lens=None):
        import torch

        return torch.tensor(self.lens if lens is None else lens, dtype=torch.int32, device="cuda")

    def hide(self, first, last, window, sinks):
        """What no query at the positions [first[s], last[s]] sees becomes NaN,
        and pages of hidden slots alone are given back."""
        st = self.pool.storage()
        for s in range(len(self.lens)):
            end = self.width * TOKENS
            seen = np.zeros(end, bool)
            if last[s] >= 0:
                seen[:min(sinks, last[s] + 1)] = True
                seen[max(0, first[s] - window + 1):last[s] + 1] = True
            for b in range(self.width):
                if self.tables[s, b] < 0:
                    continue
                here = seen[b * TOKENS:(b + 1) * TOKENS]
                if not here.any():
                    self.tables[s, b] = -1 if (s + b) % 2 else self.n_blocks + 5  # given back
                    continue
                for t in np.flatnonzero(~here):
                    poison(st, int(self.tables[s, b]), int(t), self.D, self.bits, self.mode)


def queries(seed, n, Hq, Hkv, D):
    return fast_q(seed, n, Hq, Hkv, D, outliers=False)


def window_reference(ora, oc, q, pos, window, sinks, scale):
    """f64 attention of q [Hq, D] at position pos over the oracle's stored rows."""
    if pos < 0:
        return np.zeros(q.shape)
    j = np.arange(pos + 1)
    j = j[(j < sinks) | (j > pos - window)]
    k, v = oc.dequant_kv(j)
    return ora.attention_f64(ora.bf16_to_f32(q).astype(np.float64), k, v, None, scale)


def check_window(out, ref, vmax, what=""):
    """f32 outputs: scores of soft scales stay below 64 in base 2 and come out of
    at most 32 roundings each, so they are off by 64 * 32 * 2^-24 = 2^-13 at most,
    weights and their sum by ln 2 times that each, and products with weights held
    as pairs of f16 (or bf16) by 2^-16: together below 2^-12 of the largest |V|.
    bf16 outputs: half a step of their own besides."""
    import torch

    o = out.float().cpu().numpy().astype(np.float64)
    allow = 2.0 ** -12 * vmax + (2.0 ** -8 * np.abs(ref) if out.dtype == torch.bfloat16 else 0.0)
    err = np.abs(o - ref)
    bad = ~(err <= allow)  # (a NaN is bad too)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}, "
                           f"largest {np.nanmax(err):.3e}, allowed {np.max(allow):.3e}")
