"""The operators of a paged server whose conversations share prompts and whose
caches are cut to the tokens that matter, as they are measured.

A case is a dict of plain values; `op` names the operator:

  prefix   decode attention of a batch in groups that share a long prefix (pages
           of one prompt in several block tables), the prefix once for a group
  weigh    decode attention that also adds each position's softmax weights, summed
           over the query heads, to the sequence's accumulated ones
  observe  the accumulated weights of a prompt's last queries alone
  keep     the positions that an eviction by accumulated weight keeps, with their
           weights moved along

`run` computes them with elementary torch operations, or, where `own` is true,
with the framework's calls. Both read the pages of a pool as it holds them: 16
tokens of every KV head, codes in the order of the matrix-core tiles (8 and 4
bits with an f16 scale and bias per 64 dims, in the rotated domain) or bf16 rows.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOKENS = 16  # of a page

# (KV heads, query heads, head_dim) of sliding and global layers, and of a smaller model's
SLIDING = {"Hkv": 8, "Hq": 16, "D": 256}
GLOBAL = {"Hkv": 2, "Hq": 16, "D": 512}
SMALL = {"Hkv": 4, "Hq": 8, "D": 128}


def listed():
    return [
        # two answers to one short system prompt: launch latency
        {"name": "prefix_two_a4", "op": "prefix", **SLIDING, "bits": 4, "groups": 1, "n_seqs": 2,
         "P_min": 1003, "P": 1003, "S": 40},
        # nine beams of one conversation
        {"name": "prefix_beams_a8", "op": "prefix", **GLOBAL, "bits": 8, "groups": 1, "n_seqs": 9,
         "P_min": 8000, "P": 8000, "S": 333},
        # several system prompts, their conversations ragged, unquantized
        {"name": "prefix_groups_plain", "op": "prefix", **SMALL, "bits": 16, "groups": 5, "n_seqs": 41,
         "P_min": 700, "P": 6000, "S": 500},
        # a server's decode step: 32 questions about one long document
        {"name": "prefix_batch32_a8", "op": "prefix", **GLOBAL, "bits": 8, "groups": 1, "n_seqs": 32,
         "P_min": 32768, "P": 32768, "S": 1024},
        # one token of one conversation: launch latency
        {"name": "weigh_one_a4", "op": "weigh", **SLIDING, "bits": 4, "n_seqs": 1, "T_min": 5000, "T": 5000},
        # a few conversations on a global layer, 8 bits, odd sizes
        {"name": "weigh_seven_a8", "op": "weigh", **GLOBAL, "bits": 8, "n_seqs": 7, "T_min": 37, "T": 20011},
        # a server's decode step: 32 ragged conversations
        {"name": "weigh_batch32_a4", "op": "weigh", **SLIDING, "bits": 4, "n_seqs": 32, "T_min": 512,
         "T": 16384},
        # the last questions of a short prompt, unquantized
        {"name": "observe_one_plain", "op": "observe", **SMALL, "bits": 16, "n_seqs": 1, "T_min": 3001,
         "T": 3001, "n": 5},
        # four prompts' last queries on global layers
        {"name": "observe_four_a8", "op": "observe", **GLOBAL, "bits": 8, "n_seqs": 4, "T_min": 700,
         "T": 8000, "n": 33},
        # a long prompt's last queries
        {"name": "observe_long_a4", "op": "observe", **SLIDING, "bits": 4, "n_seqs": 1, "T_min": 32768,
         "T": 32768, "n": 128},
        # one conversation cut to a budget
        {"name": "keep_one", "op": "keep", "n_seqs": 1, "T_min": 5003, "T": 5003, "most": 1024, "sinks": 4,
         "recent": 128},
        # a batch of conversations of very different lengths, the short ones whole
        {"name": "keep_batch32", "op": "keep", "n_seqs": 32, "T_min": 512, "T": 16384, "most": 4097,
         "sinks": 4, "recent": 1024},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prefix", "prefix", "weigh", "weigh", "observe", "keep"])
    shape = rng.choice([SLIDING, GLOBAL, SMALL])
    bits = rng.choice([4, 4, 8, 8, 16])
    base = {"op": op, **shape, "bits": bits}
    if op == "prefix":
        top = _log(rng, 48, 12000)
        groups = rng.choice([1, 1, 2, rng.randint(3, 6)])
        return {**base, "groups": groups, "n_seqs": groups * _log(rng, 1, 12) + rng.randint(0, 3),
                "P_min": max(1, top // rng.randint(1, 8)), "P": top, "S": _log(rng, 1, 700)}
    if op == "weigh":
        top = _log(rng, 16, 16384)
        return {**base, "n_seqs": _log(rng, 1, 16), "T_min": max(1, top // rng.randint(1, 16)), "T": top}
    if op == "observe":
        n_seqs = rng.choice([1, 1, 2, 4])
        top = _log(rng, 16, 12000)
        return {**base, "n_seqs": n_seqs, "T_min": max(1, top // rng.randint(1, 8)), "T": top,
                "n": _log(rng, 1, 160 // n_seqs)}
    top = _log(rng, 40, 32768)
    most = max(16, round(top * rng.uniform(0.03, 0.9)))
    return {"op": op, "n_seqs": _log(rng, 1, 32), "T_min": max(1, top // rng.randint(1, 16)), "T": top,
            "most": most, "sinks": rng.choice([0, rng.randint(1, 8)]), "recent": rng.randint(0, most // 2)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)


def _spread(lo, hi, n, salt):
    """n whole numbers of [lo, hi], the first the largest, the same for every seed."""
    x = np.exp(np.random.default_rng(hi * 31 + n + salt).uniform(np.log(lo), np.log(hi + 0.5), n)).astype(np.int64)
    x[0] = hi
    return x.clip(lo, hi)


def _lengths(case):
    if case["op"] != "prefix":
        return _spread(case["T_min"], case["T"], case["n_seqs"], 0)
    return _shared(case)[2] + _spread(1, case["S"], case["n_seqs"], 5)


def _shared(case):
    """Groups' first sequences (and the end), their prefixes, each sequence's prefix.
    A prefix is shared in whole pages; the last ones of a batch may be in no group."""
    g, n = case["groups"], case["n_seqs"]
    starts = np.arange(g + 1) * (n // g)
    prefix = _spread(case["P_min"], case["P"], g, 3)
    own_prefix = np.zeros(n, np.int64)
    for i in range(g):
        own_prefix[starts[i]:starts[i + 1]] = prefix[i]
    return starts, prefix, own_prefix


def _block_bytes(case):
    d, b = case["D"], case["bits"]
    return 64 * d if b == 16 else TOKENS * d * b // 4 + 2 * d


def _quantize(x, bits):
    """Codes, scale and bias (f16) of groups of 64, as the cache stores them."""
    g = x.view(*x.shape[:-1], -1, 64)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo) / (2 ** bits - 1)).clamp_min(1e-5).half()
    bias = lo.half()
    codes = ((g - bias.float()) / scale.float()).round().clamp(0, 2 ** bits - 1)
    return codes.to(torch.uint8).view(x.shape), torch.cat([scale, bias], -1)


def _nibbles(x):
    """Bytes of pairs of 4-bit codes, the first in the low half."""
    return x[..., 0::2] | x[..., 1::2] << 4


def _pages(case, n_pages, gen):
    """Pages as a pool holds them, uint8 [n_pages, Hkv, block bytes], of normal values."""
    h, d, bits = case["Hkv"], case["D"], case["bits"]
    out = torch.empty((n_pages, h, _block_bytes(case)), dtype=torch.uint8, device="cuda")
    for p0 in range(0, n_pages, 512):
        part = out[p0:p0 + 512]
        n = part.shape[0]
        k = torch.randn((n, h, TOKENS, d), generator=gen, device="cuda")
        v = torch.randn((n, h, TOKENS, d), generator=gen, device="cuda")
        if bits == 16:
            part.copy_(torch.cat([k.bfloat16().reshape(n, h, -1),
                                  v.bfloat16().transpose(2, 3).reshape(n, h, -1)], -1).view(torch.uint8))
            continue
        (kc, km), (vc, vm) = _quantize(k, bits), _quantize(v, bits)
        if bits == 8:
            kb = kc.view(n, h, 16, d // 64, 4, 16).permute(0, 1, 3, 4, 2, 5).reshape(n, h, -1)
            vb = vc.view(n, h, 4, 4, d // 64, 4, 16).permute(0, 1, 4, 2, 6, 5, 3).reshape(n, h, -1)
        else:
            kb = kc.view(n, h, 16, d // 128, 2, 2, 4, 4, 2).permute(0, 1, 3, 6, 2, 4, 5, 8, 7)
            vb = vc.view(n, h, 4, 2, 2, d // 128, 4, 2, 16).permute(0, 1, 5, 2, 8, 6, 4, 7, 3)
            kb, vb = _nibbles(kb.reshape(n, h, -1)), _nibbles(vb.reshape(n, h, -1))
        meta = [m.transpose(2, 3).reshape(n, h, -1).view(torch.uint8) for m in (km, vm)]
        part.copy_(torch.cat([kb, vb, *meta], -1))
    return out


def _tables(lens, shared, rng):
    """Shuffled pages of every sequence, those of a group's prefix the group's."""
    wide = int(max(-(-int(n) // TOKENS) for n in lens))
    table = np.full((len(lens), wide), -1, np.int32)
    order = iter(rng.permutation(sum(-(-int(n) // TOKENS) for n in lens)).astype(np.int32))
    first = np.zeros(len(lens), np.int64)  # pages that a sequence has from its group's first one
    if shared is not None:
        starts, prefix, _ = shared
        for i in range(len(prefix)):
            first[starts[i] + 1:starts[i + 1]] = prefix[i] // TOKENS
    leader = 0
    for s, n in enumerate(lens):
        if first[s] == 0:
            leader = s
        table[s, :first[s]] = table[leader, :first[s]]
        for b in range(int(first[s]), -(-int(n) // TOKENS)):
            table[s, b] = next(order)
    return table


def _pool(case, pages):
    """A pool that holds these pages."""
    fmkv = _package()
    mode = fmkv.MODE_PLAIN if case["bits"] == 16 else fmkv.MODE_AFFINE
    pool = fmkv.PagedPool(fmkv.make_desc(case["Hkv"], case["D"], case["bits"], mode=mode), pages.shape[0])
    pool.storage().copy_(pages)
    return pool


def _package():
    path = os.path.join(ROOT, "gemma4-moe-flash-mlx-turbo_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fmkv

    return fmkv


def _ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    gen, rng = _gen(seed), np.random.default_rng(seed * 131 + 11)
    lens = _lengths(case)
    st = {"case": case, "host_lens": [int(t) for t in lens], "lens": _ints(lens), "longest": int(lens.max())}
    n, wide = case["n_seqs"], int(lens.max())
    if case["op"] == "keep":
        # sums of softmax weights: a few heavy positions, many of next to nothing, some equal
        w = torch.exp(2.5 * torch.randn((n, wide), generator=gen, device="cuda")).bfloat16().float() / 64
        st["weights"] = torch.where(torch.rand((n, wide), generator=gen, device="cuda") < 0.1, 0.0, w)
        st["keep"] = torch.full((n, case["most"]), -1, dtype=torch.int32, device="cuda")
        st["n_keep"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        st["kept"] = torch.zeros((n, case["most"]), device="cuda")
        return st
    shared = _shared(case) if case["op"] == "prefix" else None
    table = _tables(lens, shared, rng)
    st["pages"] = _pages(case, int(table.max()) + 1, gen)
    st["table"], st["host_table"] = torch.from_numpy(table).cuda(), torch.from_numpy(table).long()
    hq, d = case["Hq"], case["D"]
    if case["op"] == "observe":
        # a query sees the positions up to its own; a short prompt's first ones are padding
        rows = case["n"]
        st["start"] = _ints(lens - rows)
        st["q"] = torch.randn((n, rows, hq, d), generator=gen, device="cuda").bfloat16()
    else:
        st["q"] = torch.randn((n, hq, d), generator=gen, device="cuda").bfloat16()
    if case["op"] == "prefix":
        starts, prefix, own_prefix = shared
        st["starts"], st["host_starts"] = _ints(starts), [int(x) for x in starts]
        st["prefix"], st["host_prefix"] = _ints(own_prefix), [int(x) for x in own_prefix]
        st["longest_prefix"] = int(prefix.max())
        st["longest_rest"] = int((lens - own_prefix // TOKENS * TOKENS).max())
    else:
        # what earlier steps accumulated
        st["weights"] = torch.rand((n, wide), generator=gen, device="cuda").square() * 4
        st["sums"] = torch.zeros((n, wide), device="cuda")
    st["scale"] = d ** -0.5
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own and case["op"] != "keep":
        st["pool"] = _pool(case, st.pop("pages"))
    return st


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    case = st["case"]
    if case["op"] == "prefix":
        return st["pool"].prefix_attention(st["q"], st["table"], st["lens"], st["prefix"], st["starts"],
                                           st["longest_prefix"], st["longest_rest"], scale=st["scale"])
    if case["op"] == "weigh":
        return st["pool"].weighing_attention(st["q"], st["table"], st["lens"], st["longest"], st["weights"],
                                             weights_out=st["sums"], scale=st["scale"])
    if case["op"] == "observe":
        return st["pool"].attention_weights(st["q"], st["table"], st["start"], st["longest"], st["weights"],
                                            weights_out=st["sums"], scale=st["scale"])
    return _package().heaviest_tokens(st["weights"], st["lens"], case["most"], case["sinks"], case["recent"],
                                      keep=st["keep"], n_keep=st["n_keep"], weights_out=st["kept"])


def _signs(d):
    """Signs of the cache's rotation: the top bits of a 64-bit congruential generator."""
    s, out = 42, []
    for _ in range(d):
        s = (s * 6364136223846793005 + 1442695040888963407) & (1 << 64) - 1
        out.append(-1.0 if s >> 63 else 1.0)
    return out


def _rotation(d):
    """x @ R rotates a row as the cache does before it quantizes it: Hadamard, 1 / sqrt(d), signs."""
    m = torch.ones((1, 1), device="cuda")
    while m.shape[0] < d:
        m = torch.cat([torch.cat([m, m], 1), torch.cat([m, -m], 1)], 0)
    return m * (d ** -0.5) * torch.tensor(_signs(d), device="cuda")


def _unpack(case, pages):
    """K and V of pages [n, Hkv, block bytes] as stored, f32 [Hkv, n * 16, D]."""
    n, h, d, bits = pages.shape[0], case["Hkv"], case["D"], case["bits"]
    if bits == 16:
        x = pages.view(torch.bfloat16).view(n, h, 2, TOKENS * d)
        kv = x[:, :, 0].view(n, h, TOKENS, d).float(), x[:, :, 1].view(n, h, d, TOKENS).transpose(2, 3).float()
    else:
        size = TOKENS * d * bits // 8
        kb, vb = pages[..., :size], pages[..., size:2 * size]
        meta = pages[..., 2 * size:2 * size + 2 * d].contiguous().view(torch.float16)
        meta = meta.view(n, h, 2, d // 64, TOKENS, 2).float().permute(0, 1, 2, 4, 3, 5)
        if bits == 8:
            k = kb.reshape(n, h, d // 64, 4, 16, 16).permute(0, 1, 4, 2, 3, 5)
            v = vb.reshape(n, h, d // 64, 4, 16, 4, 4).permute(0, 1, 3, 6, 2, 5, 4)
        else:
            kb, vb = (torch.stack([x & 15, x >> 4], -1) for x in (kb, vb))
            k = kb.reshape(n, h, d // 128, 4, 16, 2, 2, 2, 4).permute(0, 1, 4, 2, 5, 6, 3, 8, 7)
            v = vb.reshape(n, h, d // 128, 4, 16, 4, 2, 2, 2).permute(0, 1, 3, 8, 6, 2, 5, 7, 4)
        kv = ((x.reshape(n, h, TOKENS, d // 64, 64).float() * meta[:, :, i, :, :, :1] + meta[:, :, i, :, :, 1:])
              .reshape(n, h, TOKENS, d) for i, x in enumerate((k, v)))
    return [x.transpose(0, 1).reshape(h, n * TOKENS, d) for x in kv]


def _run_plain(st):
    case = st["case"]
    if case["op"] == "prefix":
        return _prefix_plain(st)
    if case["op"] == "weigh":
        return _weigh_plain(st)
    if case["op"] == "observe":
        return _observe_plain(st)
    return _keep_plain(st)


def _rows(st, s):
    """Query rows of sequence s by KV head, scaled (and rotated), f32 [Hkv, rows, D]."""
    case = st["case"]
    d, h, group = case["D"], case["Hkv"], case["Hq"] // case["Hkv"]
    q = st["q"][s].reshape(-1, h, group, d).transpose(0, 1).reshape(h, -1, d).float() * st["scale"]
    return q if case["bits"] == 16 else q @ st["rotation"]


def _own_pages(st, s, first, end):
    return _unpack(st["case"], st["pages"][st["host_table"][s, first:end].cuda()])


def _softmax(score):
    p = torch.exp(score - score.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _attend_plain(st, s, parts, n):
    """Output and weights of sequence s over the keys and values of `parts`, its first n."""
    q = _rows(st, s)
    score = torch.cat([torch.bmm(q, k.transpose(1, 2).contiguous()) for k, _ in parts], -1)[..., :n]
    p = _softmax(score)
    o, at = 0.0, 0
    for _, v in parts:
        part = p[..., at:at + v.shape[1]]
        o = o + torch.bmm(part, v[:, :part.shape[-1]])
        at += v.shape[1]
    if st["case"]["bits"] != 16:
        o = o @ st["rotation"].T
    return o.reshape(st["q"][s].shape).to(st["q"].dtype), p


def _prefix_plain(st):
    case = st["case"]
    st["rotation"] = _rotation(case["D"])
    out = torch.empty_like(st["q"])
    leaders = {s: e for s, e in zip(st["host_starts"], st["host_starts"][1:])}
    shared, end = None, 0
    for s, t in enumerate(st["host_lens"]):
        pages = st["host_prefix"][s] // TOKENS
        if s in leaders:
            shared, end = _own_pages(st, s, 0, pages), leaders[s]
        parts = [shared] if s < end else []
        parts.append(_own_pages(st, s, pages if s < end else 0, -(-t // TOKENS)))
        out[s] = _attend_plain(st, s, parts, t)[0]
    return out


def _weigh_plain(st):
    st["rotation"] = _rotation(st["case"]["D"])
    out, sums = torch.empty_like(st["q"]), st["sums"]
    for s, t in enumerate(st["host_lens"]):
        out[s], p = _attend_plain(st, s, [_own_pages(st, s, 0, -(-t // TOKENS))], t)
        sums[s, :t] = st["weights"][s, :t] + p.sum((0, 1))
    return out, sums


def _observe_plain(st):
    case = st["case"]
    st["rotation"] = _rotation(case["D"])
    n, group, sums = case["n"], case["Hq"] // case["Hkv"], st["sums"]
    for s, t in enumerate(st["host_lens"]):
        k = _own_pages(st, s, 0, -(-t // TOKENS))[0][:, :t]
        at = torch.arange(t - n, t, device="cuda").repeat_interleave(group)[:, None]
        score = torch.bmm(_rows(st, s), k.transpose(1, 2).contiguous())
        hidden = torch.arange(t, device="cuda") > at
        seen = at[:, 0] >= 0
        p = _softmax(score.masked_fill(hidden, -math.inf)[:, seen])
        sums[s, :t] = st["weights"][s, :t] + p.sum((0, 1))
    return sums


def _keep_plain(st):
    """The first and the last positions, and the heaviest between them, lowest index first among equals."""
    case = st["case"]
    most, sinks, recent = case["most"], case["sinks"], case["recent"]
    for s, t in enumerate(st["host_lens"]):
        w = st["weights"][s, :t]
        if t <= most:
            kept = torch.arange(t, device="cuda")
        else:
            mid = torch.sort(w[sinks:t - recent], descending=True, stable=True)[1][:most - sinks - recent]
            kept = torch.cat([torch.arange(sinks, device="cuda"), torch.sort(mid)[0] + sinks,
                              torch.arange(t - recent, t, device="cuda")])
        st["keep"][s, :len(kept)] = kept.int()
        st["n_keep"][s] = len(kept)
        st["kept"][s, :len(kept)] = w[kept]
        st["kept"][s, len(kept):] = 0.0
    return st["keep"], st["n_keep"], st["kept"]


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "keep":
        return _keep_exact(st)
    if case["op"] == "observe":
        return _observe_exact(st)
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    sums = torch.zeros(st["sums"].shape, dtype=torch.float64, device="cuda") if case["op"] == "weigh" else None
    for s, t in enumerate(st["host_lens"]):
        k, v = _rows_exact(st, s, t)
        p = torch.softmax(_scores_exact(st, st["q"][s].double(), k), -1)
        for g in range(case["Hq"]):
            out[s, g] = p[g] @ v[:, g * case["Hkv"] // case["Hq"]]
        if sums is not None:
            sums[s, :t] = st["weights"][s, :t].double() + p.sum(0)
    return out if sums is None else (out, sums)


def _places(case):
    """(byte, shift) of dim d of token t in a block's K and in its V region, numpy [2][16][D][2]."""
    d, bits = case["D"], case["bits"]
    t, x = np.meshgrid(np.arange(TOKENS), np.arange(d), indexing="ij")
    if bits == 16:
        return np.stack([np.stack([(t * d + x) * 2, 0 * t], -1), np.stack([(x * 16 + t) * 2, 0 * t], -1)])
    if bits == 8:
        k = x // 64 * 1024 + (x % 64 // 16 * 16 + t) * 16 + x % 16
        v = x // 64 * 1024 + (t // 4 * 16 + x % 16) * 16 + x % 64 // 16 * 4 + t % 4
        return np.stack([np.stack([k, 0 * t], -1), np.stack([v, 0 * t], -1)])
    o = x % 128
    nib = o % 2 * 4 + o % 8 // 2
    k = x // 128 * 1024 + (o % 32 // 8 * 16 + t) * 16 + o // 64 * 8 + o % 64 // 32 * 4 + nib // 2
    kn = nib % 2 * 4
    ct, r = o // 16, t % 4
    nib = ct % 2 * 2 + r // 2 + 4 * (r % 2)
    v = x // 128 * 1024 + (t // 4 * 16 + o % 16) * 16 + ct // 2 * 4 + nib // 2
    return np.stack([np.stack([k, kn], -1), np.stack([v, nib % 2 * 4], -1)])


def _unrotate(x):
    """Rows back from the rotated domain: signs, 1 / sqrt(d), a Hadamard product by butterflies."""
    d = x.shape[-1]
    x = x * torch.tensor(_signs(d), dtype=torch.float64, device="cuda")
    step = 1
    while step < d:
        y = x.reshape(*x.shape[:-1], d // (2 * step), 2, step)
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], -2).reshape(x.shape)
        step *= 2
    return x / math.sqrt(d)


def _rows_exact(st, s, t):
    """K and V rows of sequence s's first t positions, f64 [2, t, Hkv, D]."""
    case = st["case"]
    d, bits = case["D"], case["bits"]
    place = torch.from_numpy(_places(case)).cuda()
    pages = st["pages"][st["table"][s, :-(-t // TOKENS)].long()]
    n, rows = pages.shape[0], []
    for i in range(2):
        off = place[i, ..., 0].reshape(-1)
        if bits == 16:
            x = pages[..., i * 32 * d:(i + 1) * 32 * d].contiguous().view(torch.bfloat16)
            x = x[..., off // 2].double().view(n, -1, TOKENS, d)
        else:
            size = TOKENS * d * bits // 8
            x = pages[..., i * size:][..., off].long() >> place[i, ..., 1].reshape(-1) & 2 ** bits - 1
            meta = pages[..., 2 * size + i * d:2 * size + (i + 1) * d].contiguous().view(torch.float16).double()
            meta = meta.view(n, -1, d // 64, TOKENS, 2).repeat_interleave(64, dim=2).transpose(2, 3)
            x = _unrotate(x.view(n, -1, TOKENS, d).double() * meta[..., 0] + meta[..., 1])
        rows.append(x.permute(0, 2, 1, 3).reshape(n * TOKENS, -1, d)[:t])
    return torch.stack(rows)


def _scores_exact(st, q, k):
    """Scores of the rows q [.., Hq, D] with the keys k [t, Hkv, D], f64 [.., Hq, t]."""
    hq, h = st["case"]["Hq"], st["case"]["Hkv"]
    return torch.stack([q[..., g, :] @ k[:, g * h // hq].T.contiguous() for g in range(hq)], -2) * st["scale"]


def _observe_exact(st):
    case = st["case"]
    sums = torch.zeros(st["sums"].shape, dtype=torch.float64, device="cuda")
    for s, t in enumerate(st["host_lens"]):
        k = _rows_exact(st, s, t)[0]
        total = st["weights"][s, :t].double()
        for i in range(case["n"]):
            end = t - case["n"] + i + 1
            if end > 0:
                total[:end] += torch.softmax(_scores_exact(st, st["q"][s, i].double(), k[:end]), -1).sum(0)
        sums[s, :t] = total
    return sums


def _keep_exact(st):
    case = st["case"]
    most, sinks, recent = case["most"], case["sinks"], case["recent"]
    keep, n_keep = st["keep"].cpu().numpy().copy(), np.zeros(case["n_seqs"], np.int32)
    kept = np.zeros((case["n_seqs"], most))
    for s, t in enumerate(st["host_lens"]):
        w = st["weights"][s, :t].cpu().numpy()
        between = sorted(range(sinks, t - recent), key=lambda i: (-w[i], i))[:max(0, most - sinks - recent)]
        ids = list(range(t)) if t <= most else sorted([*range(sinks), *between, *range(t - recent, t)])
        keep[s, :len(ids)], n_keep[s], kept[s, :len(ids)] = ids, len(ids), w[ids]
    return torch.from_numpy(keep).cuda(), torch.from_numpy(n_keep).cuda(), torch.from_numpy(kept).cuda()


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _token_bytes(case):
    """K and V of one token of one KV head."""
    return 4 * case["D"] if case["bits"] == 16 else case["D"] * case["bits"] // 4 + case["D"] // 8


def work(case):
    lens = _lengths(case)
    total = int(lens.sum())
    if case["op"] == "keep":
        kept = int(np.minimum(lens, case["most"]).sum())
        return {"bytes": 4 * total + 8 * kept, "flops": total}
    h, hq, d = case["Hkv"], case["Hq"], case["D"]
    rows = 2 * len(lens) * hq * d  # bytes of q, or of the output
    if case["op"] == "prefix":
        starts, prefix, own_prefix = _shared(case)
        keys = int((prefix // TOKENS * TOKENS).sum() + (lens - own_prefix // TOKENS * TOKENS).sum())
        return {"bytes": keys * h * _token_bytes(case) + 2 * rows, "flops": 4 * hq * d * total}
    if case["op"] == "weigh":
        return {"bytes": total * (h * _token_bytes(case) + 8) + 2 * rows, "flops": 4 * hq * d * total}
    pairs = sum(int(np.maximum(np.arange(t - case["n"], t) + 1, 0).sum()) for t in lens)
    return {"bytes": total * (h * _token_bytes(case) // 2 + 8) + rows * case["n"], "flops": 2 * hq * d * pairs}
