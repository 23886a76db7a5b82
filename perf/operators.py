"""The operators a paged server needs around a layer's attention, as they are measured.

A case is a dict of plain values; `op` names the operator:

  decode   attention of one new token per sequence over a paged pool: the last
           `window` positions and the first `sinks` ones
  prefill  the same for `n` consecutive queries per sequence (a prompt chunk)
  copy     pages copied inside the pools of one or several layers (a fork's
           partly filled last pages, pages moved together)
  compact  the kept tokens of sequences moved to the front of other pages
  rope     per-head norms of q, k and v with the rotation by positions of one
           or several axes, in one pass

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
EPS = 1e-6

# (KV heads, query heads, head_dim) of sliding and global layers, and of a smaller model's
SLIDING = {"Hkv": 8, "Hq": 16, "D": 256}
GLOBAL = {"Hkv": 2, "Hq": 16, "D": 512}
SMALL = {"Hkv": 4, "Hq": 8, "D": 128}


def listed():
    return [
        # one token of one conversation on a sliding layer: launch latency
        {"name": "decode_one_a4", "op": "decode", **SLIDING, "bits": 4, "n_seqs": 1, "T_min": 5000,
         "T": 5000, "window": 1024, "sinks": 4},
        # a few conversations on a global layer kept to a window, 8 bits, odd sizes
        {"name": "decode_seven_a8", "op": "decode", **GLOBAL, "bits": 8, "n_seqs": 7, "T_min": 37,
         "T": 20011, "window": 4001, "sinks": 33},
        # a server's decode step: 32 ragged conversations, some shorter than the window
        {"name": "decode_batch32_a4", "op": "decode", **SLIDING, "bits": 4, "n_seqs": 32, "T_min": 512,
         "T": 16384, "window": 4096, "sinks": 4},
        # five drafted tokens checked after an unquantized prompt
        {"name": "prefill_five_plain", "op": "prefill", **SMALL, "bits": 16, "n_seqs": 1, "T_min": 3001,
         "T": 3001, "n": 5, "window": 1024, "sinks": 4},
        # follow-up messages of four conversations on global layers
        {"name": "prefill_four_a8", "op": "prefill", **GLOBAL, "bits": 8, "n_seqs": 4, "T_min": 700,
         "T": 8000, "n": 333, "window": 2000, "sinks": 130},
        # a prompt chunk on a sliding layer
        {"name": "prefill_chunk_a4", "op": "prefill", **SLIDING, "bits": 4, "n_seqs": 1, "T_min": 6000,
         "T": 6000, "n": 2048, "window": 1024, "sinks": 4},
        # nine beams forked: their partly filled last pages, one layer
        {"name": "copy_nine_a8", "op": "copy", **GLOBAL, "bits": 8, "layers": 1, "pages": 9},
        # a long prompt's pages moved together, the global layers of a model in one call
        {"name": "copy_many_a4", "op": "copy", **SLIDING, "bits": 4, "layers": 5, "pages": 1501},
        # one conversation of which an eviction rule keeps about a third
        {"name": "compact_one_plain", "op": "compact", **SMALL, "bits": 16, "n_seqs": 1, "T_min": 3077,
         "T": 3077, "share": 0.35},
        # a batch of conversations cut to about half, 8 bits
        {"name": "compact_eight_a8", "op": "compact", **GLOBAL, "bits": 8, "n_seqs": 8, "T_min": 3000,
         "T": 16000, "share": 0.5},
        # a decode step of 32 conversations, far positions, q, k and v of one projection
        {"name": "rope_step32", "op": "rope", **SLIDING, "n": 32, "axes": 1, "rotary": 256, "far": 131072,
         "fused": True},
        # a prompt chunk with images: three position axes, part of each head rotated
        {"name": "rope_images8k", "op": "rope", **GLOBAL, "n": 8192, "axes": 3, "rotary": 128,
         "far": 32768, "fused": False},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prefill", "prefill", "copy", "compact", "rope"])
    shape = rng.choice([SLIDING, GLOBAL, SMALL])
    bits = rng.choice([4, 4, 8, 8, 16])
    base = {"op": op, **shape}
    if op == "decode":
        n = _log(rng, 1, 16)
        top = _log(rng, 48, 16384)
        return {**base, "bits": bits, "n_seqs": n, "T_min": max(1, top // rng.randint(1, 16)), "T": top,
                "window": _log(rng, 32, 2048), "sinks": rng.choice([0, rng.randint(1, 16), _log(rng, 16, 256)])}
    if op == "prefill":
        n_seqs = rng.choice([1, 1, 2, 4])
        top = _log(rng, 16, 12000)
        return {**base, "bits": bits, "n_seqs": n_seqs, "T_min": max(1, top // rng.randint(1, 8)), "T": top,
                "n": _log(rng, 2, 1000 // n_seqs), "window": _log(rng, 32, 1024),
                "sinks": rng.choice([0, rng.randint(1, 16), _log(rng, 16, 256)])}
    if op == "copy":
        layers = rng.choice([1, 1, 2, 5])
        return {**base, "bits": bits, "layers": layers, "pages": _log(rng, 1, 1200 // layers)}
    if op == "compact":
        n = _log(rng, 1, 4)
        top = _log(rng, 40, 6000)
        return {**base, "bits": bits, "n_seqs": n, "T_min": max(1, top // rng.randint(1, 8)), "T": top,
                "share": round(rng.uniform(0.05, 0.95), 3)}
    d = shape["D"]
    axes = rng.choice([1, 1, 2, 3])
    return {**base, "n": _log(rng, 1, 6000), "axes": axes, "rotary": rng.choice([d, d, d // 2, d // 4]),
            "far": _log(rng, 64, 1 << 20), "fused": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _lengths(case):
    """Sequence lengths of [T_min, T], the first the longest, the same for every seed."""
    n = case["n_seqs"]
    rng = np.random.default_rng(case["T"] * 31 + n)
    lens = np.exp(rng.uniform(np.log(case["T_min"]), np.log(case["T"] + 0.5), n)).astype(np.int64)
    lens[0] = case["T"]
    return lens.clip(case["T_min"], case["T"])


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


def _tables(lens, first, rng, spare=0):
    """Shuffled pages for the positions [first, len) of every sequence and its
    sinks; the pages between, which a server has given back, are -1."""
    wide = int(max(-(-int(n) // TOKENS) for n in lens))
    need = [sorted({*range(0, s), *range(a, -(-int(n) // TOKENS))}) for (s, a), n in zip(first, lens)]
    total = sum(len(x) for x in need)
    order = rng.permutation(total + spare)
    table = np.full((len(lens), wide), -1, np.int32)
    at = 0
    for row, blocks in zip(table, need):
        row[blocks] = order[at:at + len(blocks)]
        at += len(blocks)
    return table, order[at:]


def _pool(case, pages):
    """A pool that holds these pages."""
    if os.path.join(ROOT, "gemma4-moe-flash-mlx-turbo_amd") not in sys.path:
        sys.path.insert(0, os.path.join(ROOT, "gemma4-moe-flash-mlx-turbo_amd"))
    import fmkv

    mode = fmkv.MODE_PLAIN if case["bits"] == 16 else fmkv.MODE_AFFINE
    pool = fmkv.PagedPool(fmkv.make_desc(case["Hkv"], case["D"], case["bits"], mode=mode), pages.shape[0])
    pool.storage().copy_(pages)
    return pool


def _inputs(case, seed):
    gen, rng = _gen(seed), np.random.default_rng(seed * 131 + 7)
    st = {"case": case}
    h, hq, d = case["Hkv"], case["Hq"], case["D"]
    if case["op"] in ("decode", "prefill"):
        n = 1 if case["op"] == "decode" else case["n"]
        lens = _lengths(case) + (n - 1)
        first = []
        for t in lens:  # pages of the sinks, first page of the window
            lo = max(0, int(t) - n + 1 - case["window"])
            first.append((min(-(-case["sinks"] // TOKENS), -(-int(t) // TOKENS)), lo // TOKENS))
        table, _ = _tables(lens, first, rng)
        st["pages"] = _pages(case, int(table.max()) + 1, gen)
        st["table"], st["host_table"] = torch.from_numpy(table).cuda(), torch.from_numpy(table).long()
        st["host_lens"] = [int(t) for t in lens]
        st["start"] = torch.tensor(lens - n, dtype=torch.int32, device="cuda")
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["longest"] = int(lens.max())
        shape = (len(lens), hq, d) if n == 1 else (len(lens), n, hq, d)
        st["q"] = torch.randn(shape, generator=gen, device="cuda").bfloat16()
        st["scale"] = d ** -0.5
    elif case["op"] == "copy":
        n = case["pages"]
        order = rng.permutation(2 * n + 3).astype(np.int32)
        st["pages"] = [_pages(case, 2 * n + 3, gen) for _ in range(case["layers"])]
        st["src"] = torch.from_numpy(order[:n]).cuda()
        st["dst"] = torch.from_numpy(order[n:2 * n]).cuda()
    elif case["op"] == "compact":
        lens = _lengths(case)
        keep = [np.sort(rng.permutation(int(t))[:round(int(t) * case["share"])]).astype(np.int32) for t in lens]
        most = max(1, max(len(k) for k in keep))
        spare = sum(-(-len(k) // TOKENS) for k in keep)
        table, free = _tables(lens, [(0, 0)] * len(lens), rng, spare)
        dst = np.full((len(lens), -(-most // TOKENS)), -1, np.int32)
        lists = np.zeros((len(lens), most), np.int32)
        for s, k in enumerate(keep):
            blocks = -(-len(k) // TOKENS)
            dst[s, :blocks], free = free[:blocks], free[blocks:]
            lists[s, :len(k)] = k
        st["pages"] = _pages(case, int(max(table.max(), dst.max())) + 1, gen)
        st["table"], st["dst"] = torch.from_numpy(table).cuda(), torch.from_numpy(dst).cuda()
        st["keep"] = torch.from_numpy(lists).cuda()
        st["host_keep"] = [len(k) for k in keep]
        st["n_keep"] = torch.tensor([len(k) for k in keep], dtype=torch.int32, device="cuda")
    else:
        n, axes = case["n"], case["axes"]
        rows = hq + 2 * h
        if case["fused"]:  # one projection's output
            x = torch.randn((n, rows, d), generator=gen, device="cuda").bfloat16()
            st["q"], st["k"], st["v"] = x[:, :hq], x[:, hq:hq + h], x[:, hq + h:]
        else:
            for name, heads in (("q", hq), ("k", h), ("v", h)):
                st[name] = torch.randn((n, heads, d), generator=gen, device="cuda").bfloat16()
        for name in ("q_weight", "k_weight"):
            st[name] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).bfloat16()
        if axes == 1 and n <= 64:  # a batch's positions, each its own
            pos = rng.integers(0, case["far"], (1, n))
        elif axes == 1:
            pos = rng.integers(0, case["far"]) + np.arange(n)[None]
        else:  # text and pictures in turn: time, then rows and columns
            i = np.arange(n)
            pos = np.stack([rng.integers(0, case["far"]) + i // 64, i // 64 + i % 64 // 8, i // 64 + i % 8])
        st["pos"] = torch.from_numpy(pos[:axes].astype(np.int32)).cuda().contiguous()
        pairs = case["rotary"] // 2
        cut = [pairs * a // axes for a in range(axes + 1)]
        st["sections"] = tuple(b - a for a, b in zip(cut, cut[1:]))
        st["theta"] = 1e6
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if not own:
        return st
    if case["op"] == "copy":
        st["pools"] = [_pool(case, p) for p in st.pop("pages")]
        st["pages"] = [p.storage() for p in st["pools"]]
    elif case["op"] == "rope":
        if os.path.join(ROOT, "gemma4-moe-flash-mlx-turbo_amd") not in sys.path:
            sys.path.insert(0, os.path.join(ROOT, "gemma4-moe-flash-mlx-turbo_amd"))
        import fmkv

        st["prologue"] = fmkv.make_qkv_prologue(st["q_weight"], st["k_weight"], EPS, case["rotary"],
                                                st["theta"], sections=st["sections"])
    else:
        st["pool"] = _pool(case, st.pop("pages"))
        st["pages"] = st["pool"].storage()
    return st


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    import fmkv

    case = st["case"]
    if case["op"] == "decode":
        return st["pool"].window_attention(st["q"], st["table"], st["lens"], st["longest"], case["window"],
                                           case["sinks"], scale=st["scale"])
    if case["op"] == "prefill":
        return st["pool"].window_prefill(st["q"], st["table"], st["start"], case["window"], case["sinks"],
                                         scale=st["scale"], max_seq_len=st["longest"])
    if case["op"] == "copy":
        fmkv.copy_blocks(st["pools"], st["src"], st["dst"])
        return [_values(case, p) for p in st["pages"]]
    if case["op"] == "compact":
        st["pool"].compact(st["table"], st["keep"], st["n_keep"], st["dst"])
        return _values(case, st["pages"])
    return fmkv.qkv_norm_rope(st["q"], st["k"], st["v"], st["pos"], st["prologue"])


def _values(case, pages):
    """Pages as an output: bf16 values, or the bytes of quantized ones, which
    move as they are and have to be equal."""
    return pages.view(torch.bfloat16) if case["bits"] == 16 else pages


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
    """K and V of pages [n, Hkv, block bytes] as stored, f32 [n, Hkv, 16, D]."""
    n, h, d, bits = pages.shape[0], case["Hkv"], case["D"], case["bits"]
    if bits == 16:
        x = pages.view(torch.bfloat16).view(n, h, 2, TOKENS * d)
        return x[:, :, 0].view(n, h, TOKENS, d).float(), x[:, :, 1].view(n, h, d, TOKENS).transpose(2, 3).float()
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
    return tuple((x.reshape(n, h, TOKENS, d // 64, 64).float() * meta[:, :, i, :, :, :1] + meta[:, :, i, :, :, 1:])
                 .reshape(n, h, TOKENS, d) for i, x in enumerate((k, v)))


def _run_plain(st):
    case = st["case"]
    if case["op"] in ("decode", "prefill"):
        return _attend_plain(st)
    if case["op"] == "copy":
        for p in st["pages"]:
            p[st["dst"].long()] = p[st["src"].long()]
        return [_values(case, p) for p in st["pages"]]
    if case["op"] == "compact":
        return _compact_plain(st)
    return _rope_plain(st)


def _attend_plain(st):
    """A sequence at a time: its visible pages, scores, softmax, products."""
    case, w, sinks = st["case"], st["case"]["window"], st["case"]["sinks"]
    d, h, group = case["D"], case["Hkv"], case["Hq"] // case["Hkv"]
    n = 1 if case["op"] == "decode" else case["n"]
    rot = _rotation(d) if case["bits"] != 16 else None
    out = torch.empty_like(st["q"])
    for s, t in enumerate(st["host_lens"]):
        lo = max(0, t - n + 1 - w) // TOKENS
        blocks = sorted({*range(0, min(-(-sinks // TOKENS), -(-t // TOKENS))), *range(lo, -(-t // TOKENS))})
        pos = (torch.tensor(blocks, device="cuda")[:, None] * TOKENS + torch.arange(TOKENS, device="cuda")).view(-1)
        k, v = _unpack(case, st["pages"][st["host_table"][s, blocks].cuda()])
        k, v = (x.transpose(0, 1).reshape(h, len(blocks) * TOKENS, d) for x in (k, v))
        q = st["q"][s].view(n, h, group, d).permute(1, 0, 2, 3).reshape(h, n * group, d).float() * st["scale"]
        if rot is not None:
            q = q @ rot
        at = torch.arange(t - n, t, device="cuda").repeat_interleave(group)[:, None]
        seen = (pos <= at) & ((pos < sinks) | (pos > at - w))
        score = torch.bmm(q, k.transpose(1, 2).contiguous()).masked_fill(~seen, -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        o = torch.bmm(p, v) / p.sum(-1, keepdim=True)
        if rot is not None:
            o = o @ rot.T
        out[s] = o.view(h, n, group, d).permute(1, 0, 2, 3).reshape(out[s].shape)
    return out


def _compact_plain(st):
    """Codes (or bf16 values) of the kept tokens taken out of their pages and put into others."""
    case, pages = st["case"], st["pages"]
    h, d, bits = case["Hkv"], case["D"], case["bits"]
    for s, n in enumerate(st["host_keep"]):
        if n == 0:
            continue
        src, dst = st["keep"][s, :n].long(), torch.arange(n, device="cuda")
        a = st["table"][s].long()[src // TOKENS], src % TOKENS
        b = st["dst"][s].long()[dst // TOKENS], dst % TOKENS
        size = TOKENS * d * bits // 8
        if bits == 16:
            x = pages.view(torch.bfloat16)
            k, v = x[..., :TOKENS * d].view(-1, h, TOKENS, d), x[..., TOKENS * d:].view(-1, h, d, TOKENS)
            k[b[0], :, b[1]] = k[a[0], :, a[1]]
            v[b[0], :, :, b[1]] = v[a[0], :, :, a[1]]
            continue
        meta = pages[..., 2 * size:].view(torch.int32).view(-1, h, 2, d // 64, TOKENS)
        meta[b[0], :, :, :, b[1]] = meta[a[0], :, :, :, a[1]]
        kb, vb = pages[..., :size], pages[..., size:2 * size]
        if bits == 8:
            k, v = kb.view(-1, h, d // 64, 4, 16, 16), vb.view(-1, h, d // 64, 4, 16, 4, 4)
            k[b[0], :, :, :, b[1]] = k[a[0], :, :, :, a[1]]
            v[b[0], :, :, b[1] // 4, :, :, b[1] % 4] = v[a[0], :, :, a[1] // 4, :, :, a[1] % 4]
            continue
        k = kb.view(-1, h, d // 128, 4, 16, 16)
        k[b[0], :, :, :, b[1]] = k[a[0], :, :, :, a[1]]
        # V: a token's nibbles, one of each byte's two, of two bytes in four
        v = vb.view(-1, h, d // 128, 4, 16, 4, 2, 2)  # [.., q, n, word, token & 1, dim tile & 1]
        t = a[1] % 4
        code = v[a[0], :, :, a[1] // 4, :, :, t % 2] >> (t // 2 * 4).to(torch.uint8).view(-1, 1, 1, 1, 1, 1) & 15
        for r in range(4):  # the four tokens that share bytes, one after the other
            m = dst % 4 == r
            i = (b[0][m], slice(None), slice(None), b[1][m] // 4, slice(None), slice(None), r % 2)
            v[i] = v[i] & (15 << 4 * (1 - r // 2)) | code[m] << 4 * (r // 2)
    return _values(case, pages)


def _rope_plain(st):
    case = st["case"]
    half = case["rotary"] // 2
    axis = torch.repeat_interleave(torch.arange(case["axes"], device="cuda"),
                                   torch.tensor(st["sections"], device="cuda"))
    freq = st["theta"] ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = st["pos"].T.double()[:, axis] * freq
    cos, sin = (f(angle).float()[:, None] for f in (torch.cos, torch.sin))
    out = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"]), (st["v"], None)):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        if w is not None:
            y = y * w.float()
            a, b = y[..., :half], y[..., half:2 * half]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], -1)
        out.append(y.bfloat16())
    return tuple(out)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] in ("decode", "prefill"):
        return _attend_exact(st)
    if case["op"] == "copy":
        done = []
        for p in st["pages"]:
            p = p.cpu().numpy()
            for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
                p[b] = p[a]
            done.append(_values(case, torch.from_numpy(p).cuda()))
        return done
    if case["op"] == "compact":
        return _compact_exact(st)
    return _rope_exact(st)


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


def _rows_exact(case, pages):
    """K and V rows of pages, f64 [2, n * 16, Hkv, D], in the rotated domain where quantized."""
    d, bits, n = case["D"], case["bits"], pages.shape[0]
    place = torch.from_numpy(_places(case)).cuda()
    rows = []
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
            x = x.view(n, -1, TOKENS, d).double() * meta[..., 0] + meta[..., 1]
        rows.append(x.permute(0, 2, 1, 3).reshape(n * TOKENS, -1, d))
    return torch.stack(rows)


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


def _attend_exact(st):
    """Every query on its own list of positions, a block of queries at a time."""
    case, w, sinks = st["case"], st["case"]["window"], st["case"]["sinks"]
    d, h, group = case["D"], case["Hkv"], case["Hq"] // case["Hkv"]
    n = 1 if case["op"] == "decode" else case["n"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    for s, t in enumerate(st["host_lens"]):
        q = st["q"][s].view(n, h, group, d).double()
        o = out[s].view(n, h, group, d)
        for i0 in range(0, n, 128):
            i1 = min(n, i0 + 128)
            first, last = t - n + i0, t - n + i1 - 1
            lo = max(0, first - w + 1)
            pos = torch.tensor(sorted({*range(0, min(sinks, last + 1)), *range(lo, last + 1)}), device="cuda")
            blk = torch.unique(pos // TOKENS)
            kv = _rows_exact(case, st["pages"][st["table"][s].long()[blk]])
            kv = kv[:, torch.searchsorted(blk, pos // TOKENS) * TOKENS + pos % TOKENS]
            if case["bits"] != 16:
                kv = _unrotate(kv)
            here = torch.arange(first, last + 1, device="cuda")
            hidden = (pos > here[:, None]) | ((pos >= sinks) & (pos <= here[:, None] - w))
            for g in range(h):
                qg = q[i0:i1, g].reshape(-1, d)
                score = (qg @ kv[0, :, g].T.contiguous()).view(i1 - i0, group, -1) * st["scale"]
                score[hidden[:, None].expand_as(score)] = -math.inf
                o[i0:i1, g] = torch.softmax(score, -1) @ kv[1, :, g].contiguous()
    return out


def _compact_exact(st):
    """Byte by byte (nibble by nibble) from the place of every dim of every token."""
    case = st["case"]
    d, bits, h = case["D"], case["bits"], case["Hkv"]
    pages = st["pages"].cpu().numpy().copy()
    place, size = _places(case), TOKENS * d * bits // 8
    table, dst, keep = (st[x].cpu().numpy() for x in ("table", "dst", "keep"))
    for s, n in enumerate(st["host_keep"]):
        for i in range(n):
            p = int(keep[s, i])
            a, b, ta, tb = pages[table[s, p // TOKENS]], pages[dst[s, i // TOKENS]], p % TOKENS, i % TOKENS
            for r in range(2):
                (fa, na), (fb, nb) = place[r, ta].T, place[r, tb].T
                fa, fb = fa + r * size, fb + r * size
                if bits == 4:
                    code = a[:, fa] >> na.astype(np.uint8) & 15
                    for half in (0, 4):
                        x = np.flatnonzero(nb == half)
                        b[:, fb[x]] = b[:, fb[x]] & (15 << 4 - half) | code[:, x] << half
                else:
                    b[:, fb] = a[:, fa]
                    if bits == 16:
                        b[:, fb + 1] = a[:, fa + 1]
                if bits != 16:
                    o = 2 * size + r * d + np.arange(d // 64)[:, None] * 64 + np.arange(4)
                    b[:, o + 4 * tb] = a[:, o + 4 * ta]
    return _values(case, torch.from_numpy(pages.reshape(-1, h, pages.shape[-1])).cuda())


def _rope_exact(st):
    case = st["case"]
    r, half = case["rotary"], case["rotary"] // 2
    pos = st["pos"].double()
    out = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"]), (st["v"], None)):
        x = x.double()
        y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
        if w is not None:
            y = y * w.double()
            z, i0 = y.clone(), 0
            for a, width in enumerate(st["sections"]):
                for i in range(i0, i0 + width):
                    phi = pos[a] * math.exp(-2 * i / r * math.log(st["theta"]))
                    c, s = torch.cos(phi)[:, None], torch.sin(phi)[:, None]
                    z[..., i] = y[..., i] * c - y[..., i + half] * s
                    z[..., i + half] = y[..., i + half] * c + y[..., i] * s
                i0 += width
            y = z
        out.append(y)
    return tuple(out)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _token_bytes(case):
    """K and V of one token of one KV head."""
    return 4 * case["D"] if case["bits"] == 16 else case["D"] * case["bits"] // 4 + case["D"] // 8


def work(case):
    h, hq, d = case["Hkv"], case["Hq"], case["D"]
    if case["op"] in ("decode", "prefill"):
        n = 1 if case["op"] == "decode" else case["n"]
        lens = _lengths(case)
        keys = pairs = 0
        for t in lens:  # (the first query's position is t - 1)
            p = np.arange(t - 1, t - 1 + n)
            lo = np.maximum(0, p + 1 - case["window"])
            sinks = np.minimum(case["sinks"], lo)
            pairs += int((p + 1 - lo + sinks).sum())
            keys += int(p[-1] + 1 - lo[0] + min(case["sinks"], lo[0]))
        return {"bytes": keys * h * _token_bytes(case) + 2 * 2 * len(lens) * n * hq * d,
                "flops": 4 * hq * d * pairs}
    if case["op"] == "copy":
        return {"bytes": 2 * case["layers"] * case["pages"] * h * _block_bytes(case), "flops": 0}
    if case["op"] == "compact":
        kept = sum(round(int(t) * case["share"]) for t in _lengths(case))
        return {"bytes": 2 * kept * h * _token_bytes(case) + 4 * kept, "flops": 0}
    rows = case["n"] * (hq + 2 * h)
    return {"bytes": 4 * rows * d + 4 * case["axes"] * case["n"], "flops": 8 * rows * d}
