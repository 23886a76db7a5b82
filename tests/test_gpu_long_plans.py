"""Calls whose plans only many or long sequences reach: first splits of four times the
others', steps of several blocks for few queries. One stored sequence, which every row of the
block tables names, each up to a length of its own."""
import numpy as np
import pytest

from gpu_util import dev_bf16, fast_kv
from shared_util import check_weights
from window_util import AFFINE, CODEBOOK, PLAIN, TOKENS, check_window, queries

pytestmark = pytest.mark.gpu

FORMS = [(m, b, D) for m, bits in ((AFFINE, (4, 8)), (CODEBOOK, (2, 3, 4)), (PLAIN, (16,))) for b in bits
         for D in (128, 256, 512)]


class Stored:
    """T tokens, the slots behind them full of NaNs; k, v: f64 rows as the oracle holds them."""

    def __init__(self, gpu, ora, mode, bits, D, Hkv, T, seed, spare=0):
        import torch

        blocks = (T + TOKENS - 1) // TOKENS
        self.pool = gpu.PagedPool(gpu.make_desc(Hkv, D, bits, mode=mode), blocks + 1 + spare)
        self.pool.storage().fill_(0xff)
        self.row = np.random.default_rng(seed).permutation(blocks + 1)[:blocks].astype(np.int32)
        self.kb, self.vb = (fast_kv(seed + i, T, Hkv, D, outliers=False) for i in (0, 5))
        oc = ora.OracleCache(Hkv, D, bits, 0, T + 1, mode=mode)
        oc.append(self.kb, self.vb)
        self.k, self.v = (torch.from_numpy(np.ascontiguousarray(x)).cuda().double() for x in oc.dequant_kv(np.arange(T)))
        self.pool.append(dev_bf16(self.kb[None]), dev_bf16(self.vb[None]), self.table(1),
                         torch.zeros(1, dtype=torch.int32, device="cuda"))

    def table(self, n):
        import torch

        return torch.from_numpy(np.tile(self.row, (n, 1))).cuda()

    def own_ends(self, lens):
        """Tables whose block of token lens[s] - 1, which a step is to store again, is a
        copy of the sequence's own (behind the first blocks + 1)."""
        import torch

        table, st = np.tile(self.row, (len(lens), 1)), self.pool.storage()
        for s, t in enumerate(lens):
            if t:
                at, mine = (t - 1) // TOKENS, len(self.row) + 1 + s
                st[mine].copy_(st[int(table[s, at])])
                table[s, at] = mine
        return torch.from_numpy(table).cuda()

    def attend(self, q, seen, scale):
        """f64 attention of q [n, G * Hkv, D], row i over the first seen[i] tokens, and the
        weights summed over the heads."""
        import torch

        n, Hq, D = q.shape
        Hkv, T = self.k.shape[1], self.k.shape[0]
        G = Hq // Hkv
        out = torch.zeros((n, Hq, D), dtype=torch.float64, device="cuda")
        total = torch.zeros((n, T), dtype=torch.float64, device="cuda")
        hidden = (torch.arange(T, device="cuda")[None] >= torch.tensor(seen, device="cuda")[:, None])[:, None]
        for h in range(Hkv):
            qh = q[:, h * G:(h + 1) * G].reshape(n * G, D).contiguous()
            s = (qh @ self.k[:, h].T.contiguous() * scale).view(n, G, T).masked_fill(hidden, -torch.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            total += p.sum(1)
            out[:, h * G:(h + 1) * G] = (p.reshape(n * G, T) @ self.v[:, h].contiguous()).view(n, G, D)
        return out.cpu().numpy(), total.cpu().numpy()


def ints(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


def lengths(n, T):
    """From none to T, and around the ends of splits of 64 blocks after a first one of 256."""
    rng = np.random.default_rng(n)
    edges = [T, T - 1, 4097, 4096, 4095, 4080, 1024, 1025, 1023, 0, 1, 16, 17]
    return (edges + [int(x) for x in rng.integers(1, T + 1, n)])[:n]


@pytest.mark.parametrize("mode,bits,D", [(AFFINE, 4, 256), (AFFINE, 8, 512), (PLAIN, 16, 128), (CODEBOOK, 3, 256),
                                         (AFFINE, 8, 128)])
def test_weighing_of_many_long_sequences(gpu, ora, mode, bits, D):
    """96 sequences of up to 6000 tokens, 8 KV heads: 288k blocks of KV heads by their bound."""
    import torch

    n, T, Hkv, Hq, scale = 96, 6000, 8, 16, D ** -0.5
    b = Stored(gpu, ora, mode, bits, D, Hkv, T, 3, spare=n)
    lens = lengths(n, T)
    qb = queries(9, n, Hq, Hkv, D)
    q = dev_bf16(qb)
    want, new = b.attend(q.double(), lens, scale)
    vmax = float(b.v.abs().max())
    old = torch.rand((n, T), generator=torch.Generator().manual_seed(2)).cuda()
    sums = torch.full((n, T), 7.0, device="cuda")
    out, _ = b.pool.weighing_attention(q, b.table(n), ints(lens), T, old, weights_out=sums, scale=scale,
                                       dtype=torch.float32)
    check_window(out, want, vmax, "output")
    before, after = old.double().cpu().numpy(), sums.double().cpu().numpy()
    for s, t in enumerate(lens):
        check_weights(after[s, :t], before[s, :t], new[s, :t], f"sequence {s} of {t}")
        assert (after[s, t:] == 7.0).all()
    # a step of the token that is stored there already
    last = [max(t - 1, 0) for t in lens]
    acc = torch.zeros((n, T), device="cuda")
    out, _ = b.pool.weighing_decode_step(
        dev_bf16(b.kb[last][:, None]), dev_bf16(b.vb[last][:, None]), b.own_ends(lens), ints([t - 1 for t in lens]),
        ints(lens), T, q, acc, scale=scale, dtype=torch.float32)
    check_window(out, want, vmax, "step")
    for s, t in enumerate(lens):
        check_weights(acc[s, :t].double().cpu().numpy(), np.zeros(t), new[s, :t], f"step, sequence {s} of {t}")
        assert not acc[s, t:].any()


@pytest.mark.parametrize("way", [1, 2, 3])
@pytest.mark.parametrize("mode,bits,D", [(AFFINE, 4, 256), (AFFINE, 8, 512), (PLAIN, 16, 128), (CODEBOOK, 3, 256)])
def test_prefixes_with_long_rests(gpu, ora, mode, bits, D, way):
    """96 sequences in three groups behind 100 tokens, the rests up to 5900 long."""
    import torch

    n, T, Hkv, Hq, scale = 96, 6000, 8, 16, D ** -0.5
    b = Stored(gpu, ora, mode, bits, D, Hkv, T, 4, spare=n)
    lens = lengths(n, T)
    q = dev_bf16(queries(19, n, Hq, Hkv, D))
    want, _ = b.attend(q.double(), lens, scale)
    vmax = float(b.v.abs().max())
    shared = (ints([min(100, t) for t in lens]), ints([0, 40, 41, n]), 100, T - 96)
    gpu.set_prefix_sharing(way)
    try:
        out = b.pool.prefix_attention(q, b.table(n), ints(lens), *shared, scale=scale, dtype=torch.float32)
        check_window(out, want, vmax, "attention")
        # (steps behind the shared blocks)
        behind = [t if t > 112 else 0 for t in lens]
        last = [max(t - 1, 0) for t in behind]
        want = np.where(np.array(behind)[:, None, None] > 0, want, 0.0)
        shared = (ints([100] * n), *shared[1:])
        out = b.pool.prefix_decode_step(
            dev_bf16(b.kb[last][:, None]), dev_bf16(b.vb[last][:, None]), b.own_ends(behind), ints([t - 1 for t in behind]),
            ints(behind), *shared, q, scale=scale, dtype=torch.float32)
        check_window(out, want, vmax, "step")
    finally:
        gpu.set_prefix_sharing(gpu.PREFIX_AUTO)


@pytest.mark.parametrize("mode,bits,D,G,n", [(*f, 2, 8) for f in FORMS] +
                         [(*f, G, n) for f in FORMS if f[2] == 128 for G, n in ((1, 13), (8, 2), (3, 5))])
def test_weights_of_few_queries_over_many_keys(gpu, ora, mode, bits, D, G, n):
    """At most 16 rows of four sequences of 4000 tokens, 8 KV heads."""
    T, Hkv, scale = 4000, 8, D ** -0.5
    lens = [T, T - 1, 3777, n - 1]
    b = Stored(gpu, ora, mode, bits, D, Hkv, T, 5)
    q = np.stack([queries(60 + s, n, Hkv * G, Hkv, D) for s in range(len(lens))])
    seen = [max(t - n + 1 + i, 0) for t in lens for i in range(n)]
    _, each = b.attend(dev_bf16(q.reshape(-1, Hkv * G, D)).double(), seen, scale)
    new = each.reshape(len(lens), n, T).sum(1)
    got = b.pool.attention_weights(dev_bf16(q), b.table(len(lens)), ints([t - n for t in lens]), T, scale=scale)
    for s, t in enumerate(lens):
        check_weights(got[s, :t].double().cpu().numpy(), np.zeros(t), new[s, :t], f"sequence {s}")
        assert not got[s, t:].any()
