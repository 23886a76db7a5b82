"""Refusals of the calls over shared prefixes, accumulated weights and kept positions."""
import ctypes

import pytest

import fmkv

BAD, NOT = fmkv.FMKV_ERR_INVALID_ARG, fmkv.FMKV_ERR_UNSUPPORTED


def test_null_pool_is_refused():
    lib = fmkv.load_library()
    calls = [
        lib.fmkv_paged_prefix_decode_attention(None, 1, 1, 4, 1, 1, 1, 1, 1, 32, 32, 8, 1.0, 1, 0, None),
        lib.fmkv_paged_prefix_decode_step(None, 1, 1, 1, 4, 1, 1, 1, 1, 1, 1, 32, 32, 1, 8, 1.0, 1, 0, None),
        lib.fmkv_paged_weighing_decode_attention(None, 1, 1, 4, 1, 1, 64, 1, 1, 64, 8, 1.0, 1, 0, None),
        lib.fmkv_paged_weighing_decode_step(None, 1, 1, 1, 4, 1, 1, 1, 64, 1, 1, 1, 64, 8, 1.0, 1, 0, None),
        lib.fmkv_paged_attention_weights(None, 1, 1, 4, 1, 1, 1, 64, 1, 1, 64, 8, 1.0, None),
    ]
    assert calls == [BAD] * len(calls)


# arguments of fmkv_heaviest_tokens, none of which may reach a launch: the addresses are none
HEAVIEST = dict(weights=1 << 20, width=64, lens=1 << 21, n=2, most=16, sinks=2, recent=4, keep=1 << 22,
                n_keep=1 << 23, out=1 << 24, out_width=16)


@pytest.mark.parametrize("change", [
    dict(n=-1), dict(n=65536), dict(width=0), dict(width=-1), dict(width=(1 << 30) + 1), dict(most=0),
    dict(most=(1 << 28) - 15), dict(sinks=-1), dict(recent=-1), dict(sinks=13), dict(recent=15),
    dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), dict(weights=None), dict(lens=None), dict(keep=None),
    dict(n_keep=None), dict(out_width=15), dict(out=1 << 20), dict(out=(1 << 20) + 508),
    dict(out=(1 << 20) - 124),
])
def test_heaviest_tokens_refuses(change):
    a = {**HEAVIEST, **change}
    rc = fmkv.load_library().fmkv_heaviest_tokens(a["weights"], a["width"], a["lens"], a["n"], a["most"], a["sinks"],
                                                  a["recent"], a["keep"], a["n_keep"], a["out"], a["out_width"], None)
    assert rc == BAD


@pytest.mark.parametrize("width", [(1 << 30) + 1, 2 ** 31 - 1])
def test_heaviest_tokens_refuses_wide_outputs(width):
    """Past the documented width (an output that is the weights: refused in any case)."""
    lib, a = fmkv.load_library(), HEAVIEST
    args = (a["weights"], a["width"], a["lens"], a["n"], a["most"], a["sinks"], a["recent"], a["keep"], a["n_keep"])
    assert lib.fmkv_heaviest_tokens(*args, a["weights"], width, None) == BAD
    assert b"kept_width" in lib.fmkv_last_error()


def test_heaviest_tokens_of_nothing():
    lib = fmkv.load_library()
    assert lib.fmkv_heaviest_tokens(None, 64, None, 0, 16, 2, 4, None, None, None, 0, None) == fmkv.FMKV_OK


@pytest.mark.parametrize("way", [-1, 4, 2 ** 31 - 1])
def test_prefix_sharing_values(way):
    with pytest.raises(fmkv.Exception_) as e:
        fmkv.set_prefix_sharing(way)
    assert e.value.code == BAD
    with pytest.raises(ValueError):
        fmkv.set_prefix_sharing(2 ** 32)
    fmkv.set_prefix_sharing(fmkv.PREFIX_AUTO)


def made(gpu, Hq=4, D=128, n=2):
    import torch

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    pool = gpu.PagedPool(gpu.make_desc(2, 128, 4), 8)
    q = torch.zeros((n, Hq, D), dtype=torch.bfloat16, device="cuda")
    return dict(pool=pool, q=q, kv=torch.zeros((n, 1, 2, 128), dtype=torch.bfloat16, device="cuda"),
                table=ints(0, 1, 2, 3, 0, 4, 5, 6).view(2, 4), lens=ints(33, 20), prefix=ints(16, 16),
                starts=ints(0, 2), out=torch.full_like(q, 7.0),
                weights=torch.full((n, 64), 7.0, dtype=torch.float32, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("change,code", [
    (dict(longest_prefix=-1), BAD), (dict(longest_rest=-1), BAD), (dict(longest_rest=65), BAD),
    (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD), (dict(Hq=3), BAD), (dict(Hq=18), NOT),
])
def test_prefix_calls_refuse(gpu, change, code):
    import torch

    a = {**dict(longest_prefix=16, longest_rest=64, scale=1.0, Hq=4), **change}
    m = made(gpu, a["Hq"])
    before = m["pool"].storage().clone()
    shared = (m["prefix"], m["starts"], a["longest_prefix"], a["longest_rest"])
    with pytest.raises(fmkv.Exception_) as e:
        m["pool"].prefix_attention(m["q"], m["table"], m["lens"], *shared, scale=a["scale"], out=m["out"])
    assert e.value.code == code
    with pytest.raises(fmkv.Exception_) as e:
        m["pool"].prefix_decode_step(m["kv"], m["kv"], m["table"], m["lens"] - 1, m["lens"], *shared, m["q"],
                                     scale=a["scale"], out=m["out"])
    assert e.value.code == code
    torch.cuda.synchronize()
    assert torch.equal(m["pool"].storage(), before) and bool((m["out"] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("change,code", [
    (dict(longest=65), BAD), (dict(longest=-1), BAD), (dict(scale=float("nan")), BAD), (dict(Hq=3), BAD),
    (dict(Hq=18), NOT),
])
def test_weighing_calls_refuse(gpu, change, code):
    import torch

    a = {**dict(longest=64, scale=1.0, Hq=4), **change}
    m = made(gpu, a["Hq"])
    before = m["pool"].storage().clone()
    kw = dict(weights_out=m["weights"], scale=a["scale"])
    for call in (lambda: m["pool"].weighing_attention(m["q"], m["table"], m["lens"], a["longest"], out=m["out"], **kw),
                 lambda: m["pool"].weighing_decode_step(m["kv"], m["kv"], m["table"], m["lens"] - 1, m["lens"],
                                                        a["longest"], m["q"], out=m["out"], **kw),
                 lambda: m["pool"].attention_weights(m["q"][:, None], m["table"], m["lens"] - 1, a["longest"], **kw)):
        with pytest.raises(fmkv.Exception_) as e:
            call()
        assert e.value.code == code
    torch.cuda.synchronize()
    assert torch.equal(m["pool"].storage(), before) and bool((m["out"] == 7.0).all())
    assert bool((m["weights"] == 7.0).all())


@pytest.mark.gpu
def test_widths_and_overlaps_are_refused(gpu):
    import torch

    m = made(gpu)
    both = torch.zeros(2 * 64 + 16, dtype=torch.float32, device="cuda")
    w = both[:128].view(2, 64)
    cases = [dict(weights_out=w[:, :32].contiguous()),              # narrower than the lengths' bound
             dict(weights=w, weights_out=both[16:].view(2, 64))]    # in part the same
    for kw in cases:
        for call in (lambda: m["pool"].weighing_attention(m["q"], m["table"], m["lens"], 64, **kw),
                     lambda: m["pool"].attention_weights(m["q"][:, None], m["table"], m["lens"] - 1, 64, **kw)):
            with pytest.raises(fmkv.Exception_) as e:
                call()
            assert e.value.code == BAD
    with pytest.raises(fmkv.Exception_) as e:
        gpu.heaviest_tokens(w, m["lens"], 16, weights_out=both[16:48].view(2, 16))
    assert e.value.code == BAD
    odd = torch.zeros(m["q"].numel() + 8, dtype=torch.bfloat16, device="cuda")[1:1 + m["q"].numel()].view(m["q"].shape)
    with pytest.raises(fmkv.Exception_) as e:
        m["pool"].prefix_attention(odd, m["table"], m["lens"], m["prefix"], m["starts"], 16, 64)
    assert e.value.code == NOT
    with pytest.raises(fmkv.Exception_) as e:
        m["pool"].weighing_attention(odd, m["table"], m["lens"], 64)
    assert e.value.code == NOT


@pytest.mark.gpu
def test_wrong_tensors_are_refused(gpu):
    m = made(gpu)
    pool, q, table, lens, prefix, starts, w = (m[k] for k in ("pool", "q", "table", "lens", "prefix", "starts", "weights"))
    good = dict(q=q, table=table, lens=lens, prefix=prefix, starts=starts)
    for change in (dict(q=q.float()), dict(q=q[..., :64].contiguous()), dict(table=table.long()), dict(lens=lens[:1]),
                   dict(lens=lens.long()), dict(prefix=prefix[:1]), dict(prefix=prefix.long()),
                   dict(starts=starts[:0]), dict(starts=starts.long()), dict(starts=starts.view(1, 2)),
                   dict(q=q.cpu()), dict(prefix=prefix.cpu()), dict(starts=starts.cpu())):
        a = {**good, **change}
        with pytest.raises(ValueError):
            pool.prefix_attention(a["q"], a["table"], a["lens"], a["prefix"], a["starts"], 16, 64)
    for bounds in ((2 ** 32 + 16, 64), (16, 2 ** 32)):
        with pytest.raises(ValueError):
            pool.prefix_attention(q, table, lens, prefix, starts, *bounds)
    for kw in (dict(weights=w.half()), dict(weights=w[:1]), dict(weights=w, weights_out=w[:, :32].contiguous()),
               dict(weights_out=w.double()), dict(weights_out=w.cpu()), dict(weights_out=w.t()),
               dict(weights_out=w[:, ::2])):
        with pytest.raises(ValueError):
            pool.weighing_attention(q, table, lens, 16, **kw)
        with pytest.raises(ValueError):
            pool.attention_weights(q[:, None], table, lens, 16, **kw)
    with pytest.raises(ValueError):
        pool.weighing_attention(q, table, lens, 2 ** 32 + 16, weights_out=w)
    for args, kw in (((w.half(), lens, 16), {}), ((w, lens.long(), 16), {}), ((w, lens, 0), {}),
                     ((w, lens, 2 ** 32 + 16), {}), ((w, lens, 16, 2 ** 32), {}), ((w.cpu(), lens, 16), {}),
                     ((w, lens, 16), dict(keep=prefix)), ((w, lens, 16), dict(n_keep=prefix[:1])),
                     ((w, lens, 16), dict(weights_out=w.half()))):
        with pytest.raises(ValueError):
            gpu.heaviest_tokens(*args, **kw)
