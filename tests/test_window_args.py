"""Refusals of the windowed calls, before any HIP call (no GPU needed)."""
import ctypes

import pytest

import fmkv


def test_null_pool_is_refused():
    lib = fmkv.load_library()
    calls = [
        lib.fmkv_paged_window_decode_attention(None, 1, 1, 4, 1, 1, 64, 8, 1.0, 16, 0, 1, 0, None),
        lib.fmkv_paged_window_decode_step(None, 1, 1, 1, 4, 1, 1, 1, 64, 1, 8, 1.0, 16, 0, 1, 0, None),
        lib.fmkv_paged_window_prefill_attention(None, 1, 1, 4, 1, 1, 4, 0, 8, 1.0, 16, 0, 1, 0, None),
        lib.fmkv_paged_window_prefill_step(None, 1, 1, 1, 4, 1, 1, 4, 0, 1, 8, 1.0, 16, 0, 1, 0, None),
        lib.fmkv_pool_storage(None, ctypes.byref(ctypes.c_void_p()), ctypes.byref(ctypes.c_int64())),
    ]
    assert calls == [fmkv.FMKV_ERR_INVALID_ARG] * len(calls)


@pytest.mark.gpu
@pytest.mark.parametrize("change,code", [
    (dict(window=0), fmkv.FMKV_ERR_INVALID_ARG), (dict(window=-1), fmkv.FMKV_ERR_INVALID_ARG),
    (dict(window=(1 << 30) + 1), fmkv.FMKV_ERR_INVALID_ARG), (dict(sinks=-1), fmkv.FMKV_ERR_INVALID_ARG),
    (dict(sinks=(1 << 30) + 1), fmkv.FMKV_ERR_INVALID_ARG), (dict(scale=float("inf")), fmkv.FMKV_ERR_INVALID_ARG),
    (dict(scale=float("nan")), fmkv.FMKV_ERR_INVALID_ARG), (dict(Hq=18), fmkv.FMKV_ERR_UNSUPPORTED),
    (dict(Hq=3), fmkv.FMKV_ERR_INVALID_ARG), (dict(max_seq_len=65), fmkv.FMKV_ERR_INVALID_ARG),
])
def test_bad_arguments_are_refused(gpu, change, code):
    import torch

    a = dict(window=16, sinks=4, scale=1.0, Hq=4, max_seq_len=64, **{})
    a.update(change)
    pool = gpu.PagedPool(gpu.make_desc(2, 128, 4), 4)
    q = torch.zeros((1, a["Hq"], 128), dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros((1, 1, 2, 128), dtype=torch.bfloat16, device="cuda")
    table = torch.zeros((1, 4), dtype=torch.int32, device="cuda")
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    before = pool.storage().clone()
    out = torch.full_like(q, 7.0)
    kw = dict(window=a["window"], sinks=a["sinks"], scale=a["scale"], out=out)
    with pytest.raises(fmkv.Exception_) as e:
        pool.window_attention(q, table, n, a["max_seq_len"], **kw)
    assert e.value.code == code
    with pytest.raises(fmkv.Exception_) as e:
        pool.window_decode_step(kv, kv, table, n - 1, n, a["max_seq_len"], q, **kw)
    assert e.value.code == code
    if "max_seq_len" not in change:
        kw["out"] = out[:, None]
        for call in (lambda: pool.window_prefill(q[:, None], table, n - 1, **kw),
                     lambda: pool.window_prefill_step(kv, kv, table, n - 1, q[:, None], **kw)):
            with pytest.raises(fmkv.Exception_) as e:
                call()
            assert e.value.code == code
    torch.cuda.synchronize()
    assert torch.equal(pool.storage(), before) and bool((out == 7.0).all())


@pytest.mark.gpu
def test_wrong_tensors_are_refused(gpu):
    import torch

    pool = gpu.PagedPool(gpu.make_desc(2, 128, 4), 4)
    q = torch.zeros((1, 4, 128), dtype=torch.bfloat16, device="cuda")
    table = torch.zeros((1, 4), dtype=torch.int32, device="cuda")
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    for bad in ((q.float(), table, n), (q[..., :64].contiguous(), table, n), (q, table.long(), n),
                (q, table.repeat(2, 1), n), (q, table, n.repeat(2)), (q, table, n.long()), (q.cpu(), table, n)):
        with pytest.raises(ValueError):
            pool.window_attention(*bad, 64, 16)
    with pytest.raises(ValueError):
        pool.window_attention(q, table, n, 64, 16, out=torch.zeros((1, 4, 64), device="cuda"))
    for window, sinks in ((2 ** 32 + 16, 0), (16, 2 ** 32)):
        for call in (lambda: pool.window_attention(q, table, n, 64, window, sinks),
                     lambda: pool.window_prefill(q[:, None], table, n - 1, window, sinks)):
            with pytest.raises(ValueError):
                call()
    off = torch.zeros(q.numel() + 8, dtype=torch.bfloat16, device="cuda")[1:1 + q.numel()].view(q.shape)
    with pytest.raises(fmkv.Exception_) as e:
        pool.window_attention(off, table, n, 64, 16)
    assert e.value.code == fmkv.FMKV_ERR_UNSUPPORTED


@pytest.mark.parametrize("wide", [2 ** 32 + 16, 2 ** 31, -2 ** 31 - 1, 16 - 2 ** 32, 2 ** 64 + 16])
def test_lengths_past_32_bits_are_refused(wide):
    """A bound of 2^32 + 16 would arrive as 16, and decode leave out what splits for 16
    positions do not cover. In every call that takes one, before any HIP call."""
    import torch

    pool = object.__new__(fmkv.PagedPool)
    pool.desc, pool._lib, pool._h, pool._D, pool._H, pool._device = fmkv.make_desc(2, 128, 4), None, None, 128, 2, -1
    q, kv = (torch.zeros((1, 1, h, 128), dtype=torch.bfloat16) for h in (4, 2))
    table, n = torch.zeros((1, 4), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    pro = fmkv.KvPrologue()
    for call in (lambda: pool.window_attention(q[0], table, n, wide, 16),
                 lambda: pool.window_decode_step(kv, kv, table, n, n, wide, q[0], 16),
                 lambda: pool.window_prefill(q, table, n, 16, max_seq_len=wide),
                 lambda: pool.window_prefill_step(kv, kv, table, n, q, 16, max_seq_len=wide),
                 lambda: pool.attention(q[0], table, n, wide),
                 lambda: pool.decode_step(kv, kv, table, n, n, wide, q[0]),
                 lambda: pool.decode_step_projected(kv, kv, table, n, n, wide, pro, q[0]),
                 lambda: pool.prefill_step(kv, kv, table, n, q, max_seq_len=wide)):
        with pytest.raises(ValueError, match="max_seq_len does not fit"):
            call()


@pytest.mark.parametrize("wide", [2 ** 32 + 16, -2 ** 32 + 16])
def test_descriptions_and_prologues_past_32_bits_are_refused(wide):
    for change in ("n_kv_heads", "head_dim", "bits", "window", "mode", "group_size"):
        with pytest.raises(ValueError, match=change):
            fmkv.make_desc(**{**dict(n_kv_heads=2, head_dim=128, bits=4), change: wide})
    with pytest.raises(ValueError, match="rope_dims"):
        fmkv.make_qkv_prologue(None, None, 1e-6, wide, 1e4)
    with pytest.raises(ValueError, match="section"):
        fmkv.make_qkv_prologue(None, None, 1e-6, 64, 1e4, sections=(16, wide))
