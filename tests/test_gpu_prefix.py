"""Decode attention of batches that share prefixes, against 64-bit references
over each sequence's own rows."""
import numpy as np
import pytest

from gpu_util import check_codes, dev_bf16, fast_kv
from shared_util import Shared, attend_reference, poison_from
from window_util import AFFINE, CODEBOOK, PLAIN, TOKENS, check_window, queries

pytestmark = pytest.mark.gpu

WAYS = ["alone", "rows", "tiles"]


@pytest.fixture
def way(request, gpu):
    gpu.set_prefix_sharing(1 + WAYS.index(request.param))
    yield request.param
    gpu.set_prefix_sharing(gpu.PREFIX_AUTO)


every_way = pytest.mark.parametrize("way", WAYS, indirect=True)

# mode, bits, D, Hkv, Hq
FORMS = [(AFFINE, 4, 256, 8, 16), (AFFINE, 8, 512, 2, 16), (PLAIN, 16, 128, 4, 8), (AFFINE, 4, 128, 2, 2),
         (AFFINE, 8, 256, 1, 5), (AFFINE, 4, 512, 1, 8), (AFFINE, 8, 128, 3, 9), (CODEBOOK, 2, 128, 2, 4),
         (CODEBOOK, 3, 256, 2, 12), (CODEBOOK, 4, 512, 1, 7), (CODEBOOK, 3, 512, 2, 2), (PLAIN, 16, 512, 1, 8),
         (PLAIN, 16, 256, 2, 6), (CODEBOOK, 4, 256, 1, 1), (CODEBOOK, 3, 128, 2, 16)]

# groups of (prefix, lengths), the sequences of no group before and after
BATCHES = {
    "pair": ([(160, [171, 200])], ((), ())),
    # a prefix that ends inside a block, members at its very end, inside it, of no length
    "edges": ([(77, [77, 64, 90, 0, 79, 17, 1, 80, 100])], ((5,), (33, 0))),
    # lone sequences as groups, one shorter than a block, an empty group, a prefix of nothing
    "lone": ([(40, [55]), (9, [25, 26]), (300, [300]), (0, [31]), (48, [])], ((), (1,))),
    # more sequences than a tile holds at any number of heads, uneven groups
    "many": ([(513, list(range(514, 514 + 70))), (35, [36] * 3), (128, [129 + 7 * i for i in range(20)])], ((), ())),
    "long": ([(3001, [3010, 3500, 3001]), (1600, [1601, 1700])], ((), (700,))),
}


def reference(ora, b, q, scale):
    return np.stack([attend_reference(ora, oc, q[s], n, scale)[0] for s, (oc, n) in enumerate(zip(b.oracles, b.lens))])


def vmax(b):
    return max(float(np.abs(oc.dequant_kv(np.arange(n))[1]).max()) for oc, n in zip(b.oracles, b.lens) if n)


@every_way
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", FORMS)
def test_attention(gpu, ora, mode, bits, D, Hkv, Hq, batch, way):
    import torch

    groups, alone = BATCHES[batch]
    b = Shared(gpu, ora, mode, D, bits, Hkv, groups, alone, seed=3)
    q = queries(11, len(b.lens), Hq, Hkv, D)
    want = reference(ora, b, q, D ** -0.5)
    big = vmax(b)
    tables, lens, prefix, starts, longest, rest = b.args()
    # the tight bounds, and looser ones: more ranges of keys, most of them of none
    for dtype, bound in ((torch.float32, longest), (torch.bfloat16, longest), (torch.float32, longest + 9000),
                         (torch.float32, 2 ** 31 - 1)):
        out = b.pool.prefix_attention(dev_bf16(q), tables, lens, prefix, starts, bound, rest, scale=D ** -0.5,
                                      dtype=dtype)
        check_window(out, want, big, f"{batch} {dtype} {bound}")


def test_bounds_of_two_billion(gpu, ora):
    """A batch that reads its own tables, wide enough for bounds whose sum 32 bits do not hold."""
    import torch

    b = Shared(gpu, ora, AFFINE, 128, 4, 1, [(40, [50])], seed=25)
    q = queries(43, 1, 1, 1, 128)
    tables, lens, prefix, starts, longest, rest = b.args()
    wide = torch.zeros((1, 1 << 28), dtype=torch.int32, device="cuda")
    wide[:, :tables.shape[1]] = tables
    want = reference(ora, b, q, 128 ** -0.5)
    for bounds in ((longest, rest), (2 ** 31 - 1, rest), (2 ** 31 - 1, 2 ** 31 - 1)):
        out = b.pool.prefix_attention(dev_bf16(q), wide, lens, prefix, starts, *bounds, scale=128 ** -0.5,
                                      dtype=torch.float32)
        check_window(out, want, vmax(b), f"{bounds}")


@every_way
@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", [FORMS[0], FORMS[2], FORMS[7]])
def test_more_groups_than_lanes(gpu, ora, mode, bits, D, Hkv, Hq, way):
    """Groups are looked through 64 at a time."""
    import torch

    groups = [(33 + i % 3 * 16, [50 + i % 3 * 16 + j for j in range(1 + i % 4)]) for i in range(131)]
    b = Shared(gpu, ora, mode, D, bits, Hkv, groups, ((20,), (9,)), seed=21)
    q = queries(41, len(b.lens), Hq, Hkv, D)
    out = b.pool.prefix_attention(dev_bf16(q), *b.args(), scale=D ** -0.5, dtype=torch.float32)
    check_window(out, reference(ora, b, q, D ** -0.5), vmax(b), "many groups")


def test_automatic(gpu, ora):
    """The choice by sizes, from two sequences to many behind a long prefix."""
    import torch

    for Hkv, Hq, D in ((8, 16, 256), (2, 16, 512)):
        for prefix, n in ((20, 2), (640, 3), (640, 40), (5000, 4), (5000, 33)):
            b = Shared(gpu, ora, AFFINE, D, 4, Hkv, [(prefix, [prefix + 1 + 3 * i for i in range(n)])], seed=15)
            q = dev_bf16(queries(23, n, Hq, Hkv, D))
            got = b.pool.prefix_attention(q, *b.args(), scale=D ** -0.5, dtype=torch.float32)
            want = b.pool.window_attention(q, b.table(), b.ints(b.lens), max(b.lens), window=2 ** 30, scale=D ** -0.5,
                                           dtype=torch.float32)
            # (two results, each within the bound of check_window)
            check_window(got, want.double().cpu().numpy(), 2 * vmax(b), f"{n} behind {prefix}")


@every_way
@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", FORMS)
def test_step(gpu, ora, mode, bits, D, Hkv, Hq, way):
    """Three steps of one token per sequence, a padded row among them; stored codes
    bit for bit; the shared blocks as they were."""
    import torch

    b = Shared(gpu, ora, mode, D, bits, Hkv, [(77, [77, 80, 95, 101]), (32, [32, 47])], ((6,), (0,)), seed=5, room=4)
    n = len(b.lens)
    padded = 3  # a row of no sequence: length 0, position -1
    for step in range(3):
        k, v = (fast_kv(500 + 10 * step + i, n, Hkv, D, outliers=False) for i in (0, 1))
        q = queries(60 + step, n, Hq, Hkv, D)
        shared = b.pool.storage()[torch.from_numpy(b.tables[1, :4]).long().cuda()].clone()
        lens = [t + 1 for t in b.lens]
        lens[padded] = 0
        start = [t - 1 for t in lens]
        for s in range(n):
            if s != padded:
                b.oracles[s].append(k[s:s + 1], v[s:s + 1])
                b.lens[s] += 1
        rest = max(t - min(p, t) // TOKENS * TOKENS if b.starts[0] <= s < b.starts[-1] else t
                   for s, (t, p) in enumerate(zip(b.lens, b.prefix)))
        out = b.pool.prefix_decode_step(
            dev_bf16(k[:, None]), dev_bf16(v[:, None]), b.table(), b.ints(start), b.ints(lens), b.ints(b.prefix),
            b.ints(b.starts), max(b.prefix), rest, dev_bf16(q), scale=D ** -0.5, dtype=torch.float32)
        want = reference(ora, b, q, D ** -0.5)
        want[padded] = 0.0
        check_window(out, want, vmax(b), f"step {step}")
        assert not out[padded].any()
        assert torch.equal(b.pool.storage()[torch.from_numpy(b.tables[1, :4]).long().cuda()], shared)
    codes, meta = b.pool.read_codes()
    for s in range(n):
        at = np.arange(b.lens[s])
        slots = torch.from_numpy(b.tables[s, at // TOKENS] * TOKENS + at % TOKENS).long().cuda()
        check_codes(codes[slots], meta[slots], b.oracles[s], slots=at, what=f"sequence {s}")


@every_way
@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", [FORMS[0], FORMS[1], FORMS[2], FORMS[8]])
def test_hidden_slots(gpu, ora, mode, bits, D, Hkv, Hq, way):
    """What lies past a sequence's length, in its blocks and in the shared ones, does
    not reach its output."""
    import torch

    b = Shared(gpu, ora, mode, D, bits, Hkv, [(160, [180, 175, 160])], ((), (20,)), seed=7)
    q = queries(13, 4, Hq, Hkv, D)
    tables, lens, prefix, starts, longest, rest = b.args()
    # a member that sees 37 of the shared positions, where the others' rows are infinite
    short = b.ints([180, 37, 160, 20])
    before = b.pool.prefix_attention(dev_bf16(q), tables, short, prefix, starts, longest, rest, scale=D ** -0.5,
                                     dtype=torch.float32)
    poison_from(b, 0, 40)
    after = b.pool.prefix_attention(dev_bf16(q), tables, short, prefix, starts, longest, rest, scale=D ** -0.5,
                                    dtype=torch.float32)
    want = attend_reference(ora, b.oracles[1], q[1], 37, D ** -0.5)[0]
    check_window(after[1:2], want[None], vmax(b), "the short member")
    assert torch.equal(after[3], before[3])
    assert not torch.equal(after[0], before[0])  # (which sees them)


def not_finite_but_where_the_formula_is(out, kind, what):
    """out: results that a value of `kind` goes into: that infinity, or NaN."""
    o = out.cpu().numpy()
    assert not np.isfinite(o).any(), what
    assert (np.isnan(o) | (o == kind)).all(), f"{what}: {o[~(np.isnan(o) | (o == kind))]}"


@every_way
@pytest.mark.parametrize("D,Hkv,Hq", [(128, 4, 8), (512, 1, 8), (256, 2, 6)])
def test_values_that_are_not_finite(gpu, ora, D, Hkv, Hq, way):
    """bf16 values of either sign that are not finite, in blocks that every row sees and
    in ones that a member does not see whole: the members that see them have that
    infinity or NaN in that dim, the others and the other dims what they had."""
    import torch

    b = Shared(gpu, ora, PLAIN, D, 16, Hkv, [(160, [180, 175, 160])], ((), (20,)), seed=7)
    q = queries(13, 4, Hq, Hkv, D)
    tables, lens, prefix, starts, longest, rest = b.args()
    short = b.ints([180, 37, 160, 20])
    args = (dev_bf16(q), tables, short, prefix, starts, longest, rest)
    before = b.pool.prefix_attention(*args, scale=D ** -0.5, dtype=torch.float32)
    st = b.pool.storage()
    bad = {5: (-np.inf, 0xff80), 9: (np.nan, 0x7fc0), 11: (np.inf, 0x7f80), 70: (np.nan, 0xffff)}
    for d, (_, bits) in bad.items():
        token = 38 + d % 3  # (past the short member's, in the block that it sees in part)
        o = 32 * D + d * 2 * TOKENS + 2 * (token % TOKENS)
        block = st[int(b.tables[0, token // TOKENS])]
        block[:, o], block[:, o + 1] = bits & 255, bits >> 8
    after = b.pool.prefix_attention(*args, scale=D ** -0.5, dtype=torch.float32)
    rest_dims = [d for d in range(D) if d not in bad]
    assert torch.equal(after[3], before[3])
    check_window(after[1:2], attend_reference(ora, b.oracles[1], q[1], 37, D ** -0.5)[0][None], vmax(b), "the short member")
    for s in (0, 2):
        assert torch.equal(after[s][:, rest_dims], before[s][:, rest_dims])
        for d, (kind, _) in bad.items():
            not_finite_but_where_the_formula_is(after[s, :, d], kind, f"sequence {s}, {kind}")


@pytest.mark.parametrize("window", [0, 100])
def test_prefill_values_that_are_not_finite(gpu, ora, window):
    """The same of a chunk's queries."""
    import torch

    D, Hkv, Hq, prefix, n = 128, 2, 4, 20, 150
    book = Shared(gpu, ora, PLAIN, D, 16, Hkv, [(0, [prefix + n])], seed=9)
    q = dev_bf16(np.stack([queries(300 + i, 1, Hq, Hkv, D)[0] for i in range(n)])[None])
    start = book.ints([prefix])
    st = book.pool.storage()
    for kind, bits in ((-np.inf, 0xff80), (np.nan, 0x7fc0), (np.inf, 0x7f80)):
        token, d = 56, 7
        o = 32 * D + d * 2 * TOKENS + 2 * (token % TOKENS)
        block = st[int(book.tables[0, token // TOKENS])]
        block[:, o], block[:, o + 1] = bits & 255, bits >> 8
        out = book.pool.window_prefill(q, book.table(), start, window or 2 ** 30, scale=D ** -0.5, dtype=torch.float32)[0]
        sees = np.arange(prefix, prefix + n)
        sees = (sees >= token) & (sees < token + (window or 2 ** 30))
        assert torch.isfinite(out[torch.from_numpy(~sees).cuda()]).all()
        others = [x for x in range(D) if x != d]
        assert torch.isfinite(out[:, :, others]).all()
        not_finite_but_where_the_formula_is(out[torch.from_numpy(sees).cuda()][:, :, d], kind, f"{kind}")


@every_way
@pytest.mark.parametrize("mode,bits,D,Hkv,Hq", [(CODEBOOK, 4, 128, 2, 6), (CODEBOOK, 2, 256, 1, 3), (CODEBOOK, 2, 512, 1, 2)])
def test_other_codebooks(gpu, ora, mode, bits, D, Hkv, Hq, way):
    """The widths that are not among the forms above, over slots full of NaNs."""
    for batch in BATCHES:
        test_attention(gpu, ora, mode, bits, D, Hkv, Hq, batch, way)
    test_step(gpu, ora, mode, bits, D, Hkv, Hq, way)
    test_hidden_slots(gpu, ora, mode, bits, D, Hkv, Hq, way)


@every_way
def test_graph_and_streams(gpu, ora, way):
    """A captured step replayed with eager calls between, on tensors of another
    stream; the same bits each time."""
    import torch

    D, Hkv, Hq = 256, 8, 16
    b = Shared(gpu, ora, AFFINE, D, 4, Hkv, [(400, [410 + i for i in range(9)])], seed=9)
    q = dev_bf16(queries(17, 9, Hq, Hkv, D))
    args = b.args()
    want = b.pool.prefix_attention(q, *args, scale=D ** -0.5)
    other = torch.cuda.Stream()
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.pool.prefix_attention(q, *args, scale=D ** -0.5, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(b.pool.prefix_attention(q, *args, scale=D ** -0.5), want)
        torch.cuda.synchronize()
    got = b.pool.prefix_attention(q, *args, scale=D ** -0.5, stream=other)
    other.synchronize()
    assert torch.equal(got, want)


@every_way
def test_forked_book(gpu, ora, way):
    """The blocks that PageBook.fork shares, as a server uses them: the same
    attention as over each sequence's whole table."""
    import torch

    D, Hkv, Hq, bits, prompt = 512, 2, 16, 8, 203
    book = gpu.PageBook(64)
    pool = gpu.PagedPool(gpu.make_desc(Hkv, D, bits), 64)
    parent = book.alloc(-(-prompt // TOKENS))
    k, v = (dev_bf16(fast_kv(i, prompt, Hkv, D, outliers=False)[None]) for i in (1, 2))
    table = torch.tensor([parent], dtype=torch.int32, device="cuda")
    pool.append(k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    rows, copies = [parent], []
    for _ in range(4):
        child, copy = book.fork(parent, prompt)
        rows.append(child)
        copies.append(copy)
    src, dst = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*copies))
    gpu.copy_blocks([pool], src, dst)
    rows = [r + book.alloc(1) for r in rows]
    tables = torch.tensor(rows, dtype=torch.int32, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    n = len(rows)
    for step in range(8):
        kn, vn = (dev_bf16(fast_kv(40 + 2 * step + i, n, Hkv, D, outliers=False)[:, None]) for i in (0, 1))
        q = dev_bf16(queries(80 + step, n, Hq, Hkv, D))
        t = prompt + step + 1
        out = pool.prefix_decode_step(kn, vn, tables, ints([t - 1] * n), ints([t] * n), ints([prompt] * n),
                                      ints([0, n]), prompt, t - prompt // TOKENS * TOKENS, q, scale=D ** -0.5,
                                      dtype=torch.float32)
        want = pool.window_attention(q, tables, ints([t] * n), t, window=2 ** 30, scale=D ** -0.5,
                                     dtype=torch.float32)
        check_window(out, want.double().cpu().numpy(), 2 * float(vn.abs().max() + v.abs().max()), f"step {step}")
