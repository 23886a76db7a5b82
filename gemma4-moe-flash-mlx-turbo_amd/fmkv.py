"""Python host binding of the fmkv C ABI (include/fmkv.h).

Mirrors the reference's Rust cache API (src/cache.rs:186-310) so callers and
tests read like the reference:

    cache = KVCache.new_quantized_with_window(head_dim=256, bits=4, window=1024,
                                              n_kv_heads=8)
    cache.update_and_fetch(k, v)          # append (store half); returns a view
    out = cache.attention(q, scale=1.0)   # decode read (SDPA replacement)
    cache.offset(), cache.stored_len(), cache.peek_kv()

Device memory and streams come from PyTorch (plumbing only): tensors are
passed to the library as raw device pointers. The HIP library is required;
nothing here computes on the CPU, and loading fails loudly when libfmkv.so is
missing.
"""
from __future__ import annotations

import contextlib
import ctypes
import os
from dataclasses import dataclass
from pathlib import Path

import torch  # imported before libfmkv.so so both share torch's HIP runtime

PKG_DIR = Path(__file__).resolve().parent
LIB_PATH = PKG_DIR / "libfmkv.so"

FMKV_OK = 0
FMKV_ERR_INVALID_ARG = 1
FMKV_ERR_UNSUPPORTED = 2
FMKV_ERR_OOM = 3
FMKV_ERR_HIP = 4
FMKV_ERR_CAPACITY = 5
MODE_AFFINE = 0
MODE_CODEBOOK = 1
MODE_PLAIN = 2  # unquantized bf16 rows (bits 16): KVCacheInner::Plain, src/cache.rs:174-178
PLAIN_BITS = 16
PREFIX_AUTO, PREFIX_ALONE, PREFIX_ROWS, PREFIX_TILES = 0, 1, 2, 3  # see set_prefix_sharing
DTYPE_BF16 = 0
DTYPE_F32 = 1
BLOCK_TOKENS = 16

EXPORTED = (
    "fmkv_last_error", "fmkv_validate_desc", "fmkv_layout_bytes", "fmkv_cache_create",
    "fmkv_cache_destroy", "fmkv_cache_offset", "fmkv_cache_stored_len", "fmkv_cache_append",
    "fmkv_cache_trim", "fmkv_decode_attention", "fmkv_cache_fetch", "fmkv_cache_read_codes",
    "fmkv_pool_create", "fmkv_pool_destroy", "fmkv_paged_append", "fmkv_paged_decode_attention",
    "fmkv_cache_append_projected", "fmkv_paged_append_projected",
    "fmkv_pool_read_codes", "fmkv_set_blocks_per_split", "fmkv_set_sparse_v_gather",
    "fmkv_cache_decode_splits",
    "fmkv_profile_enable", "fmkv_profile_collect", "fmkv_profile_collect_each",
    "fmkv_decode_step", "fmkv_paged_decode_step",
    "fmkv_prefill_step", "fmkv_paged_prefill_step", "fmkv_paged_prefill_step_bounded",
    "fmkv_decode_step_noalloc",
    "fmkv_decode_step_projected", "fmkv_paged_decode_step_projected",
    "fmkv_paged_window_decode_attention", "fmkv_paged_window_decode_step",
    "fmkv_paged_window_prefill_attention", "fmkv_paged_window_prefill_step", "fmkv_pool_storage",
    "fmkv_pools_copy_blocks", "fmkv_paged_compact", "fmkv_qkv_norm_rope",
    "fmkv_paged_prefix_decode_attention", "fmkv_paged_prefix_decode_step",
    "fmkv_paged_weighing_decode_attention", "fmkv_paged_weighing_decode_step",
    "fmkv_paged_attention_weights", "fmkv_heaviest_tokens", "fmkv_set_prefix_sharing",
    "fmkv_pages_create", "fmkv_pages_destroy", "fmkv_pages_free_count", "fmkv_pages_users",
    "fmkv_pages_alloc", "fmkv_pages_release", "fmkv_pages_fork", "fmkv_pages_slide",
)


class Exception_(RuntimeError):
    """Error raised for a non-zero fmkv status (mirrors mlx_rs::error::Exception)."""

    def __init__(self, code: int, msg: str):
        super().__init__(f"fmkv error {code}: {msg}")
        self.code = code


class CacheDesc(ctypes.Structure):
    _fields_ = [
        ("n_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("bits", ctypes.c_int32),
        ("group_size", ctypes.c_int32),
        ("mode", ctypes.c_int32),
        ("window", ctypes.c_int32),
        ("capacity", ctypes.c_int64),
        ("sign_seed", ctypes.c_uint64),
    ]


class KvPrologue(ctypes.Structure):
    """fmkv_kv_prologue: the layer's k_norm / v_norm / RoPE fused into the
    append (src/model/gemma4_attention.rs:52-81)."""
    _fields_ = [
        ("k_norm_weight", ctypes.c_void_p),
        ("eps", ctypes.c_float),
        ("rope_dims", ctypes.c_int32),
        ("rope_theta", ctypes.c_float),
        ("v_from_k", ctypes.c_int32),
    ]


def make_prologue(k_norm_weight: torch.Tensor, eps: float, rope_dims: int, rope_theta: float,
                  v_from_k: bool = False) -> KvPrologue:
    """k_norm_weight: bf16 [head_dim] on the device. The struct holds a
    reference to the tensor, so the weight lives as long as the prologue
    (the C struct itself carries only the device address)."""
    if k_norm_weight.dtype != torch.bfloat16 or k_norm_weight.dim() != 1:
        raise ValueError("k_norm_weight must be bf16 [head_dim]")
    if not k_norm_weight.is_contiguous() or not k_norm_weight.is_cuda:
        raise ValueError("k_norm_weight must be contiguous and on the GPU")
    _check_bits("rope_dims", rope_dims, 32)
    pro = KvPrologue(k_norm_weight.data_ptr(), eps, rope_dims, rope_theta, 1 if v_from_k else 0)
    pro.weight = k_norm_weight
    return pro


def _check_prologue_weight(prologue: KvPrologue, head_dim: int, keys: torch.Tensor) -> None:
    """The weight is of the head's length and on the GPU of the rows."""
    w = getattr(prologue, "weight", None)
    if w is None:
        return
    if w.numel() != head_dim:
        raise ValueError(f"k_norm_weight has {w.numel()} elements; head_dim is {head_dim}")
    if w.get_device() != keys.get_device():
        raise ValueError(f"k_norm_weight is on {w.device}, the rows are on {keys.device}")


class QkvPrologue(ctypes.Structure):
    """fmkv_qkv_prologue: the norms of q, k and v and the rotation of q and k
    (src/model/gemma4_attention.rs:50-81), see qkv_norm_rope."""
    _fields_ = [
        ("q_norm_weight", ctypes.c_void_p),
        ("k_norm_weight", ctypes.c_void_p),
        ("eps", ctypes.c_float),
        ("rope_dims", ctypes.c_int32),
        ("rope_theta", ctypes.c_float),
        ("n_axes", ctypes.c_int32),
        ("sections", ctypes.c_int32 * 4),
        ("v_norm", ctypes.c_int32),
        ("v_from_k", ctypes.c_int32),
    ]


def make_qkv_prologue(q_norm_weight, k_norm_weight, eps: float, rope_dims: int, rope_theta: float,
                      sections=None, v_norm: bool = True, v_from_k: bool = False) -> QkvPrologue:
    """Weights bf16 [head_dim] on the device (None for rows that are never
    given); sections: pairs of each position axis (None: one axis). The struct
    keeps the weights alive, as make_prologue's does."""
    for w in (q_norm_weight, k_norm_weight):
        if w is not None and (w.dtype != torch.bfloat16 or w.dim() != 1 or not w.is_contiguous() or
                              not w.is_cuda):
            raise ValueError("norm weights must be contiguous bf16 [head_dim] on the GPU")
    cut = tuple(sections) if sections is not None else (rope_dims // 2,)
    if not 1 <= len(cut) <= 4:
        raise ValueError("sections must be one to four counts of pairs")
    for name, value in (("rope_dims", rope_dims), *(("a section", x) for x in cut)):
        _check_bits(name, value, 32)
    pro = QkvPrologue(None if q_norm_weight is None else q_norm_weight.data_ptr(),
                      None if k_norm_weight is None else k_norm_weight.data_ptr(), eps, rope_dims,
                      rope_theta, len(cut), (ctypes.c_int32 * 4)(*cut), int(v_norm), int(v_from_k))
    pro.weights = (q_norm_weight, k_norm_weight)
    return pro


_lib = None


def load_library(path: str | os.PathLike | None = None) -> ctypes.CDLL:
    """Load libfmkv.so (built by build.py); raises if it is missing."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise RuntimeError(
            f"{p} not found: build the HIP library first (python {PKG_DIR / 'build.py'})")
    lib = ctypes.CDLL(str(p))
    vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
    P = ctypes.POINTER
    sig = {
        "fmkv_last_error": ([], ctypes.c_char_p),
        "fmkv_validate_desc": ([P(CacheDesc)], ctypes.c_int),
        "fmkv_layout_bytes": ([P(CacheDesc), P(i64), P(i64)], ctypes.c_int),
        "fmkv_cache_create": ([P(CacheDesc), P(vp)], ctypes.c_int),
        "fmkv_cache_destroy": ([vp], ctypes.c_int),
        "fmkv_cache_offset": ([vp, P(i64)], ctypes.c_int),
        "fmkv_cache_stored_len": ([vp, P(i64)], ctypes.c_int),
        "fmkv_cache_append": ([vp, vp, vp, i64, vp], ctypes.c_int),
        "fmkv_cache_trim": ([vp, i64], ctypes.c_int),
        "fmkv_decode_attention": ([vp, vp, i32, ctypes.c_float, ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_cache_fetch": ([vp, vp, vp, i32, vp], ctypes.c_int),
        "fmkv_cache_read_codes": ([vp, vp, vp, vp], ctypes.c_int),
        "fmkv_pool_create": ([P(CacheDesc), i64, P(vp)], ctypes.c_int),
        "fmkv_pool_destroy": ([vp], ctypes.c_int),
        "fmkv_paged_append": ([vp, vp, vp, vp, i32, vp, i32, i32, vp], ctypes.c_int),
        "fmkv_cache_append_projected": ([vp, vp, vp, i64, P(KvPrologue), vp], ctypes.c_int),
        "fmkv_paged_append_projected": ([vp, vp, vp, vp, i32, vp, i32, i32, P(KvPrologue), vp],
                                        ctypes.c_int),
        "fmkv_paged_decode_attention": ([vp, vp, vp, i32, vp, i32, i32, i32, ctypes.c_float,
                                         ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_pool_read_codes": ([vp, vp, vp, vp], ctypes.c_int),
        "fmkv_set_blocks_per_split": ([i32], ctypes.c_int),
        "fmkv_set_sparse_v_gather": ([i32], ctypes.c_int),
        "fmkv_set_prefix_sharing": ([i32], ctypes.c_int),
        "fmkv_cache_decode_splits": ([vp, P(i32)], ctypes.c_int),
        "fmkv_profile_enable": ([i32], ctypes.c_int),
        "fmkv_profile_collect": ([P(ctypes.c_double), P(i32)], ctypes.c_int),
        "fmkv_profile_collect_each": ([P(ctypes.c_float), i32, P(i32)], ctypes.c_int),
        "fmkv_decode_step": ([vp, vp, vp, i64, vp, i32, ctypes.c_float, ctypes.c_float, vp, i32,
                              vp], ctypes.c_int),
        "fmkv_decode_step_noalloc": ([vp, vp, vp, i64, vp, i32, ctypes.c_float, ctypes.c_float, vp,
                                      i32, vp], ctypes.c_int),
        "fmkv_prefill_step": ([vp, vp, vp, i64, vp, i32, ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_prefill_step": ([vp, vp, vp, vp, i32, vp, i32, i32, vp, i32, ctypes.c_float, vp,
                                     i32, vp], ctypes.c_int),
        "fmkv_paged_prefill_step_bounded": ([vp, vp, vp, vp, i32, vp, i32, i32, i32, vp, i32,
                                             ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_decode_step": ([vp, vp, vp, vp, i32, vp, vp, i32, i32, i32, vp, i32,
                                    ctypes.c_float, ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_decode_step_projected": ([vp, vp, vp, i64, P(KvPrologue), vp, i32, ctypes.c_float,
                                        ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_decode_step_projected": ([vp, vp, vp, vp, i32, vp, vp, i32, i32, i32,
                                              P(KvPrologue), vp, i32, ctypes.c_float,
                                              ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_window_decode_attention": ([vp, vp, vp, i32, vp, i32, i32, i32, ctypes.c_float,
                                                i32, i32, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_window_decode_step": ([vp, vp, vp, vp, i32, vp, vp, i32, i32, vp, i32,
                                           ctypes.c_float, i32, i32, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_window_prefill_attention": ([vp, vp, vp, i32, vp, i32, i32, i32, i32,
                                                 ctypes.c_float, i32, i32, vp, i32, vp],
                                                ctypes.c_int),
        "fmkv_paged_window_prefill_step": ([vp, vp, vp, vp, i32, vp, i32, i32, i32, vp, i32,
                                            ctypes.c_float, i32, i32, vp, i32, vp], ctypes.c_int),
        "fmkv_pool_storage": ([vp, P(vp), P(i64)], ctypes.c_int),
        "fmkv_pools_copy_blocks": ([P(vp), i32, vp, vp, i64, vp], ctypes.c_int),
        "fmkv_paged_compact": ([vp, vp, i32, vp, i32, vp, vp, i32, i32, vp], ctypes.c_int),
        "fmkv_qkv_norm_rope": ([P(QkvPrologue), i32, i32, i32, i64, vp, i64, vp, i64, vp, i64, vp,
                                vp, vp, vp, vp], ctypes.c_int),
        "fmkv_paged_prefix_decode_attention": ([vp, vp, vp, i32, vp, i32, vp, vp, i32, i32, i32, i32,
                                                ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_prefix_decode_step": ([vp, vp, vp, vp, i32, vp, vp, i32, vp, vp, i32, i32, i32,
                                           vp, i32, ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_weighing_decode_attention": ([vp, vp, vp, i32, vp, i32, i32, vp, vp, i32, i32,
                                                  ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_weighing_decode_step": ([vp, vp, vp, vp, i32, vp, vp, i32, i32, vp, vp, vp, i32,
                                             i32, ctypes.c_float, vp, i32, vp], ctypes.c_int),
        "fmkv_paged_attention_weights": ([vp, vp, vp, i32, vp, i32, i32, i32, vp, vp, i32, i32,
                                          ctypes.c_float, vp], ctypes.c_int),
        "fmkv_heaviest_tokens": ([vp, i32, vp, i32, i32, i32, i32, vp, vp, vp, i32, vp],
                                 ctypes.c_int),
        "fmkv_pages_create": ([i64, P(vp)], ctypes.c_int),
        "fmkv_pages_destroy": ([vp], ctypes.c_int),
        "fmkv_pages_free_count": ([vp, P(i64)], ctypes.c_int),
        "fmkv_pages_users": ([vp, i32, P(i32)], ctypes.c_int),
        "fmkv_pages_alloc": ([vp, i64, P(i32)], ctypes.c_int),
        "fmkv_pages_release": ([vp, P(i32), i64], ctypes.c_int),
        "fmkv_pages_fork": ([vp, P(i32), i64, P(i32), P(i32), P(i32)], ctypes.c_int),
        "fmkv_pages_slide": ([vp, P(i32), i64, i32, i32, P(i64)], ctypes.c_int),
    }
    for name, (args, res) in sig.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    if path is None:
        _lib = lib
    return lib


def _check(rc: int) -> None:
    if rc != FMKV_OK:
        raise Exception_(rc, load_library().fmkv_last_error().decode())


def _ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("fmkv needs device tensors")
    if not t.is_contiguous():
        raise ValueError("fmkv needs contiguous tensors")
    return t.data_ptr()


def _here(t: torch.Tensor | None, device: int) -> int | None:
    """_ptr of a tensor that has to be on GPU `device`."""
    if t is None:
        return None
    if t.get_device() != device:
        raise ValueError(f"fmkv needs tensors on cuda:{device}, got one on {t.device}")
    if not t.is_contiguous():
        raise ValueError("fmkv needs contiguous tensors")
    return t.data_ptr()


def _on(stream):
    """Where an output is allocated that a call on `stream` writes (None: the
    current stream), so that torch does not reuse memory that another stream
    still works on."""
    if stream is None:
        return contextlib.nullcontext()
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream))
    return torch.cuda.stream(stream)


# The current stream's handle alone: making a torch.cuda.Stream takes longer than a
# launch. (Not a public name of torch's: where it is missing, the public way.)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream) -> int | None:
    if stream is None:
        if _raw_stream is None:
            return torch.cuda.current_stream().cuda_stream
        return _raw_stream(torch.cuda.current_device())
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def make_desc(n_kv_heads: int, head_dim: int, bits: int, window: int = 0, capacity: int = 0,
              mode: int = MODE_AFFINE, group_size: int = 64, sign_seed: int = 42) -> CacheDesc:
    for name, value in (("n_kv_heads", n_kv_heads), ("head_dim", head_dim), ("bits", bits),
                        ("group_size", group_size), ("mode", mode), ("window", window)):
        _check_bits(name, value, 32)
    _check_bits("capacity", capacity, 64)
    return CacheDesc(n_kv_heads, head_dim, bits, group_size, mode, window, capacity, sign_seed)


def validate(desc: CacheDesc) -> None:
    _check(load_library().fmkv_validate_desc(ctypes.byref(desc)))


def layout_bytes(desc: CacheDesc) -> tuple[int, int]:
    b, a = ctypes.c_int64(), ctypes.c_int64()
    _check(load_library().fmkv_layout_bytes(ctypes.byref(desc), ctypes.byref(b), ctypes.byref(a)))
    return b.value, a.value


def set_blocks_per_split(bps: int) -> None:
    """Blocks per split-K work-group for decode attention (0: the plan's);
    a paged sequence's first split takes 4 x bps blocks when the grid holds
    at least four work-groups per CU."""
    _check(load_library().fmkv_set_blocks_per_split(bps))


def set_sparse_v_gather(on: bool) -> None:
    """Sparse-V after its statistics pass: the gather of the kept V rows
    (True, the default) or the gated pass and the split merge (False)."""
    _check(load_library().fmkv_set_sparse_v_gather(1 if on else 0))


def set_prefix_sharing(way: int) -> None:
    """How batches that share prefixes run: PREFIX_AUTO (by a call's sizes), or always
    each sequence alone, eight rows at a time, or 64 (for tuning and tests)."""
    _check_bits("way", way, 32)
    _check(load_library().fmkv_set_prefix_sharing(way))


def profile_enable(max_records: int) -> None:
    """Record HIP events around the next max_records split-K kernels."""
    _check(load_library().fmkv_profile_enable(max_records))


def profile_collect() -> tuple[float, int]:
    """(summed kernel milliseconds, launches timed) since the last collect."""
    ms, n = ctypes.c_double(), ctypes.c_int32()
    _check(load_library().fmkv_profile_collect(ctypes.byref(ms), ctypes.byref(n)))
    return ms.value, n.value


def profile_collect_each(capacity: int) -> list[float]:
    """Kernel milliseconds of each launch timed since the last collect."""
    buf, n = (ctypes.c_float * max(capacity, 1))(), ctypes.c_int32()
    _check(load_library().fmkv_profile_collect_each(buf, capacity, ctypes.byref(n)))
    return [buf[i] for i in range(n.value)]


class KVCache:
    """KV cache of one attention layer (src/cache.rs:166-172): quantized
    (affine or codebook) or plain bf16."""

    def __init__(self, desc: CacheDesc):
        self.desc = desc
        self._lib = load_library()
        h = ctypes.c_void_p()
        _check(self._lib.fmkv_cache_create(ctypes.byref(desc), ctypes.byref(h)))
        self._h = h

    # --- constructors mirroring src/cache.rs:202-227 --------------------------
    @classmethod
    def new_quantized_with_window(cls, head_dim: int, bits: int, window: int | None,
                                  n_kv_heads: int, capacity: int = 0,
                                  mode: int = MODE_AFFINE, sign_seed: int = 42) -> "KVCache":
        return cls(make_desc(n_kv_heads, head_dim, bits, window or 0, capacity, mode,
                             sign_seed=sign_seed))

    @classmethod
    def new_quantized(cls, head_dim: int, bits: int, n_kv_heads: int, capacity: int,
                      mode: int = MODE_AFFINE) -> "KVCache":
        return cls.new_quantized_with_window(head_dim, bits, None, n_kv_heads, capacity, mode)

    @classmethod
    def new_with_window(cls, head_dim: int, window: int | None, n_kv_heads: int,
                        capacity: int = 0) -> "KVCache":
        """The plain bf16 cache (KVCache::new_with_window, src/cache.rs:191-199)."""
        return cls(make_desc(n_kv_heads, head_dim, PLAIN_BITS, window or 0, capacity, MODE_PLAIN))

    @classmethod
    def new(cls, head_dim: int, n_kv_heads: int, capacity: int) -> "KVCache":
        """KVCache::new (src/cache.rs:187-189): plain, no window."""
        return cls.new_with_window(head_dim, None, n_kv_heads, capacity)

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.fmkv_cache_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # --- state (src/cache.rs:229-242) ------------------------------------------
    def offset(self) -> int:
        v = ctypes.c_int64()
        _check(self._lib.fmkv_cache_offset(self._h, ctypes.byref(v)))
        return v.value

    def stored_len(self) -> int:
        v = ctypes.c_int64()
        _check(self._lib.fmkv_cache_stored_len(self._h, ctypes.byref(v)))
        return v.value

    # --- append / fetch (src/cache.rs:247-310) ---------------------------------
    def append(self, keys: torch.Tensor, values: torch.Tensor, stream=None) -> None:
        """keys/values: bf16 [n_tokens, n_kv_heads, head_dim] on the device."""
        self._check_kv(keys, values)
        _check(self._lib.fmkv_cache_append(self._h, _ptr(keys), _ptr(values), keys.shape[0],
                                           _stream(stream)))

    def append_projected(self, keys: torch.Tensor, values: torch.Tensor | None,
                         prologue: KvPrologue, stream=None) -> None:
        """append() of raw k_proj / v_proj rows through the layer's prologue
        (k_norm + RoPE on K, v_norm on V; values None with prologue.v_from_k)."""
        if values is None:
            values = keys
        self._check_kv(keys, values)
        _check_prologue_weight(prologue, self.desc.head_dim, keys)
        _check(self._lib.fmkv_cache_append_projected(self._h, _ptr(keys), _ptr(values),
                                                     keys.shape[0], ctypes.byref(prologue),
                                                     _stream(stream)))

    def update_and_fetch(self, keys: torch.Tensor, values: torch.Tensor, stream=None,
                         fetch: bool = False):
        """Store new positions; with fetch=True also return the visible
        dequantized K/V like the reference's return value."""
        self.append(keys, values, stream)
        return self.peek_kv(stream=stream) if fetch else None

    def peek_kv(self, dtype=torch.bfloat16, stream=None):
        n = self.stored_len()
        if n == 0:
            return None
        shape = (n, self.desc.n_kv_heads, self.desc.head_dim)
        k = torch.empty(shape, dtype=dtype, device="cuda")
        v = torch.empty(shape, dtype=dtype, device="cuda")
        _check(self._lib.fmkv_cache_fetch(self._h, _ptr(k), _ptr(v), _dtype_code(dtype),
                                          _stream(stream)))
        return k, v

    def trim(self, keep_last: int) -> None:
        _check(self._lib.fmkv_cache_trim(self._h, keep_last))

    # --- attention read (src/model/gemma4_attention.rs:94-103) -----------------
    def attention(self, q: torch.Tensor, scale: float = 1.0, sparse_v_tau: float = 0.0,
                  out: torch.Tensor | None = None, dtype=torch.bfloat16, stream=None) -> torch.Tensor:
        """q: bf16 [n_q_heads, head_dim] -> out [n_q_heads, head_dim]."""
        if q.dtype != torch.bfloat16 or q.dim() != 2 or q.shape[1] != self.desc.head_dim:
            raise ValueError("q must be bf16 [n_q_heads, head_dim]")
        if out is None:
            out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(self._lib.fmkv_decode_attention(self._h, _ptr(q), q.shape[0], scale, sparse_v_tau,
                                               _ptr(out), _dtype_code(out.dtype), _stream(stream)))
        return out

    def decode_step(self, keys: torch.Tensor, values: torch.Tensor, q: torch.Tensor,
                    scale: float = 1.0, sparse_v_tau: float = 0.0, out: torch.Tensor | None = None,
                    dtype=torch.bfloat16, stream=None) -> torch.Tensor:
        """update_and_fetch(keys, values) then attention(q) in one call
        (src/model/gemma4_attention.rs:84-103); shapes as append / attention."""
        self._check_kv(keys, values)
        if q.dtype != torch.bfloat16 or q.dim() != 2 or q.shape[1] != self.desc.head_dim:
            raise ValueError("q must be bf16 [n_q_heads, head_dim]")
        if out is None:
            out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(self._lib.fmkv_decode_step(self._h, _ptr(keys), _ptr(values), keys.shape[0],
                                          _ptr(q), q.shape[0], scale, sparse_v_tau, _ptr(out),
                                          _dtype_code(out.dtype), _stream(stream)))
        return out

    def decode_step_projected(self, keys: torch.Tensor, values: torch.Tensor | None,
                              prologue: KvPrologue, q: torch.Tensor, scale: float = 1.0,
                              sparse_v_tau: float = 0.0, out: torch.Tensor | None = None,
                              dtype=torch.bfloat16, stream=None) -> torch.Tensor:
        """decode_step() of raw k_proj / v_proj rows through the layer's
        prologue (src/model/gemma4_attention.rs:50-104 after the projections;
        values None with prologue.v_from_k)."""
        if values is None:
            values = keys
        self._check_kv(keys, values)
        _check_prologue_weight(prologue, self.desc.head_dim, keys)
        if q.dtype != torch.bfloat16 or q.dim() != 2 or q.shape[1] != self.desc.head_dim:
            raise ValueError("q must be bf16 [n_q_heads, head_dim]")
        if out is None:
            out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(self._lib.fmkv_decode_step_projected(
            self._h, _ptr(keys), _ptr(values), keys.shape[0], ctypes.byref(prologue), _ptr(q),
            q.shape[0], scale, sparse_v_tau, _ptr(out), _dtype_code(out.dtype), _stream(stream)))
        return out

    def prefill_step(self, keys: torch.Tensor, values: torch.Tensor, q: torch.Tensor,
                     scale: float = 1.0, out: torch.Tensor | None = None, dtype=torch.bfloat16,
                     stream=None) -> torch.Tensor:
        """update_and_fetch of an L-token chunk and the chunk's causal (sliding:
        banded) attention (src/model/gemma4_attention.rs:84-104 with L > 1,
        masks src/model/mod.rs:682-753). keys/values bf16 [L, n_kv_heads, D];
        q bf16 [L, n_q_heads, D]; returns [L, n_q_heads, D]."""
        self._check_kv(keys, values)
        if (q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[0] != keys.shape[0]
                or q.shape[2] != self.desc.head_dim):
            raise ValueError("q must be bf16 [n_tokens, n_q_heads, head_dim]")
        if out is None:
            out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(self._lib.fmkv_prefill_step(self._h, _ptr(keys), _ptr(values), keys.shape[0],
                                           _ptr(q), q.shape[1], scale, _ptr(out),
                                           _dtype_code(out.dtype), _stream(stream)))
        return out

    def decode_splits(self) -> int:
        v = ctypes.c_int32()
        _check(self._lib.fmkv_cache_decode_splits(self._h, ctypes.byref(v)))
        return v.value

    # --- raw contents for bit-exact checks -------------------------------------
    def n_slots(self) -> int:
        """Stored slots: a ring's window rounded up to whole 16-token blocks,
        or a linear cache's capacity."""
        w = self.desc.window
        return (w + 15) // 16 * 16 if w > 0 else self.desc.capacity

    def read_codes(self, stream=None):
        """(codes uint32 [n_slots, 2, H, words], meta uint16 [n_slots, 2, H, n_meta])."""
        return _read_codes(self._lib.fmkv_cache_read_codes, self._h, self.desc, self.n_slots(), stream)

    def _check_kv(self, keys, values):
        d = self.desc
        for t in (keys, values):
            if t.dtype != torch.bfloat16 or t.dim() != 3 or t.shape[1:] != (d.n_kv_heads, d.head_dim):
                raise ValueError(f"K/V must be bf16 [n, {d.n_kv_heads}, {d.head_dim}], got "
                                 f"{tuple(t.shape)} {t.dtype}")
        if keys.shape != values.shape:
            raise ValueError("keys and values differ in shape")


@dataclass(frozen=True)
class LayerCacheSpec:
    """One layer's cache shape as Model::make_cache derives it
    (src/model/mod.rs:375-396 with the per-layer dims of :448-465)."""
    is_full: bool     # layer_types[i] == "full_attention"
    use_k_eq_v: bool  # attention_k_eq_v && is_full
    head_dim: int     # global_head_dim on full layers, else head_dim
    n_kv_heads: int   # num_global_key_value_heads on K==V layers
    window: int       # sliding_window on layers that are not K==V, else 0
    bits: int


def layer_cache_specs(layer_types, head_dim: int, n_kv_heads: int, *,
                      global_head_dim: int | None = None, n_global_kv_heads: int | None = None,
                      sliding_window: int | None = None, attention_k_eq_v: bool = False,
                      kv_quant_bits: int = 3, global_kv_quant_bits: int | None = None):
    """Per-layer cache shapes of a Gemma-4 stack, the choices of
    Model::make_cache (src/model/mod.rs:375-396) and the layer constructor
    (:448-465): a layer is full iff its type is "full_attention"; K==V
    layers are the full ones when attention_k_eq_v; only layers that are
    not K==V get the sliding window (so with attention_k_eq_v false every
    layer does, as in the reference); full layers use global_head_dim
    (default head_dim); K==V layers use n_global_kv_heads (default
    n_kv_heads). kv_quant_bits applies to every layer unless
    global_kv_quant_bits overrides it on full layers (a mixed 4/8-bit
    stack)."""
    specs = []
    for t in layer_types:
        is_full = t == "full_attention"
        k_eq_v = bool(attention_k_eq_v and is_full)
        specs.append(LayerCacheSpec(
            is_full, k_eq_v,
            (global_head_dim or head_dim) if is_full else head_dim,
            (n_global_kv_heads or n_kv_heads) if k_eq_v else n_kv_heads,
            0 if k_eq_v or not sliding_window else int(sliding_window),
            global_kv_quant_bits if (is_full and global_kv_quant_bits) else kv_quant_bits))
    return specs


def make_cache(layer_types, head_dim: int, n_kv_heads: int, *, capacity: int,
               global_head_dim: int | None = None, n_global_kv_heads: int | None = None,
               sliding_window: int | None = None, attention_k_eq_v: bool = False,
               kv_quant_bits: int | None = 3, global_kv_quant_bits: int | None = None,
               mode: int = MODE_CODEBOOK, sign_seed: int = 42) -> list:
    """One cache per layer, as Model::make_cache (src/model/mod.rs:375-396)
    builds them with KVCache::new_quantized_with_window(layer.kv_head_dim(),
    bits, window). The reference's quantized cache is the TurboQuant
    codebook (default 3 bits, src/main.rs:82-84), hence mode's default;
    MODE_AFFINE gives the 4/8-bit affine caches. `capacity` bounds the
    positions of the linear (window 0) caches, whose arenas are
    preallocated. kv_quant_bits None gives the reference's plain bf16
    caches (KVCache::new_with_window, --no-kv-quant) on every layer."""
    plain = kv_quant_bits is None
    specs = layer_cache_specs(layer_types, head_dim, n_kv_heads, global_head_dim=global_head_dim,
                              n_global_kv_heads=n_global_kv_heads, sliding_window=sliding_window,
                              attention_k_eq_v=attention_k_eq_v,
                              kv_quant_bits=PLAIN_BITS if plain else kv_quant_bits,
                              global_kv_quant_bits=None if plain else global_kv_quant_bits)
    caches = []
    for sp in specs:
        if plain:
            c = KVCache.new_with_window(sp.head_dim, sp.window or None, sp.n_kv_heads,
                                        capacity=0 if sp.window else capacity)
        else:
            c = KVCache.new_quantized_with_window(sp.head_dim, sp.bits, sp.window or None,
                                                  sp.n_kv_heads, capacity=0 if sp.window else capacity,
                                                  mode=mode, sign_seed=sign_seed)
        c.spec = sp
        caches.append(c)
    return caches


class PagedPool:
    """Pool of 16-token blocks shared by many sequences (batched decode)."""

    def __init__(self, desc: CacheDesc, n_blocks: int):
        _check_bits("n_blocks", n_blocks, 64)
        self.desc = desc
        self.n_blocks = n_blocks
        self._D, self._H = desc.head_dim, desc.n_kv_heads  # (a struct's field takes longer to read)
        self._lib = load_library()
        h = ctypes.c_void_p()
        _check(self._lib.fmkv_pool_create(ctypes.byref(desc), n_blocks, ctypes.byref(h)))
        self._h = h
        self._device = torch.cuda.current_device()

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.fmkv_pool_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def append(self, keys, values, block_tables, start_pos, stream=None) -> None:
        """keys/values bf16 [n_seqs, n_new, H, D]; block_tables int32 [n_seqs, max_blocks];
        start_pos int32 [n_seqs]."""
        n_seqs, n_new = keys.shape[0], keys.shape[1]
        _check(self._lib.fmkv_paged_append(self._h, _ptr(keys), _ptr(values), _ptr(block_tables),
                                           block_tables.shape[1], _ptr(start_pos), n_seqs, n_new,
                                           _stream(stream)))

    def append_projected(self, keys, values, block_tables, start_pos, prologue: KvPrologue,
                         stream=None) -> None:
        """append() of raw projections through the layer's prologue."""
        if values is None:
            values = keys
        n_seqs, n_new = keys.shape[0], keys.shape[1]
        _check_prologue_weight(prologue, self.desc.head_dim, keys)
        _check(self._lib.fmkv_paged_append_projected(
            self._h, _ptr(keys), _ptr(values), _ptr(block_tables), block_tables.shape[1],
            _ptr(start_pos), n_seqs, n_new, ctypes.byref(prologue), _stream(stream)))

    def prefill_step(self, keys, values, block_tables, start_pos, q, scale: float = 1.0,
                     out=None, dtype=torch.bfloat16, stream=None, max_seq_len: int = 0):
        """append(keys, values, ...) at start_pos, then each sequence's causal
        attention of its n_new queries. keys/values bf16 [n_seqs, n_new,
        n_kv_heads, D]; q bf16 [n_seqs, n_new, n_q_heads, D]. max_seq_len: the
        longest sequence's length after the call, where the host knows it (for
        speed only, on tables wider than that; 0: the table's width)."""
        if q.dim() != 4 or q.shape[:2] != keys.shape[:2]:
            raise ValueError("q must be bf16 [n_seqs, n_new, n_q_heads, head_dim]")
        _check_bits("max_seq_len", max_seq_len, 32)
        if out is None:
            out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(self._lib.fmkv_paged_prefill_step_bounded(
            self._h, _ptr(keys), _ptr(values), _ptr(block_tables), block_tables.shape[1],
            _ptr(start_pos), keys.shape[0], keys.shape[1], max_seq_len, _ptr(q), q.shape[2], scale,
            _ptr(out), _dtype_code(out.dtype), _stream(stream)))
        return out

    def attention(self, q, block_tables, seq_lens, max_seq_len: int, scale: float = 1.0,
                  sparse_v_tau: float = 0.0, out=None, dtype=torch.bfloat16, stream=None):
        """q bf16 [n_seqs, n_q_heads, D]; seq_lens int32 [n_seqs]."""
        _check_bits("max_seq_len", max_seq_len, 32)
        if out is None:
            out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(self._lib.fmkv_paged_decode_attention(
            self._h, _ptr(q), _ptr(block_tables), block_tables.shape[1], _ptr(seq_lens),
            q.shape[0], max_seq_len, q.shape[1], scale, sparse_v_tau, _ptr(out),
            _dtype_code(out.dtype), _stream(stream)))
        return out

    def decode_step(self, keys, values, block_tables, start_pos, seq_lens, max_seq_len: int, q,
                    scale: float = 1.0, sparse_v_tau: float = 0.0, out=None, dtype=torch.bfloat16,
                    stream=None):
        """append(keys, values, ...) at start_pos, then attention over seq_lens
        (= start_pos + n_new) in one call."""
        _check_bits("max_seq_len", max_seq_len, 32)
        if out is None:
            out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(self._lib.fmkv_paged_decode_step(
            self._h, _ptr(keys), _ptr(values), _ptr(block_tables), block_tables.shape[1],
            _ptr(start_pos), _ptr(seq_lens), keys.shape[0], keys.shape[1], max_seq_len, _ptr(q),
            q.shape[1], scale, sparse_v_tau, _ptr(out), _dtype_code(out.dtype), _stream(stream)))
        return out

    def decode_step_projected(self, keys, values, block_tables, start_pos, seq_lens,
                              max_seq_len: int, prologue: KvPrologue, q, scale: float = 1.0,
                              sparse_v_tau: float = 0.0, out=None, dtype=torch.bfloat16,
                              stream=None):
        """decode_step() of raw projections through the layer's prologue
        (RoPE positions from start_pos; values None with prologue.v_from_k)."""
        if values is None:
            values = keys
        _check_prologue_weight(prologue, self.desc.head_dim, keys)
        _check_bits("max_seq_len", max_seq_len, 32)
        if out is None:
            out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(self._lib.fmkv_paged_decode_step_projected(
            self._h, _ptr(keys), _ptr(values), _ptr(block_tables), block_tables.shape[1],
            _ptr(start_pos), _ptr(seq_lens), keys.shape[0], keys.shape[1], max_seq_len,
            ctypes.byref(prologue), _ptr(q), q.shape[1], scale, sparse_v_tau, _ptr(out),
            _dtype_code(out.dtype), _stream(stream)))
        return out

    def window_attention(self, q, block_tables, seq_lens, max_seq_len: int, window: int,
                         sinks: int = 0, scale: float = 1.0, out=None, dtype=torch.bfloat16,
                         stream=None):
        """attention() of each sequence's newest token over its last `window`
        positions and its first `sinks` ones. q bf16 [n_seqs, n_q_heads, D];
        seq_lens int32 [n_seqs]. Pages that hold neither are not looked up."""
        n, heads, _ = _check_tensor("q", q, torch.bfloat16, (None, None, self._D))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        _check_tensor("seq_lens", seq_lens, torch.int32, (n,))
        _check_window(window, sinks, max_seq_len)
        dev = self._device
        out = _out(out, q, dtype, stream)
        _check(self._lib.fmkv_paged_window_decode_attention(
            self._h, _here(q, dev), _here(block_tables, dev), width, _here(seq_lens, dev), n,
            max_seq_len, heads, scale, window, sinks, _here(out, dev), _dtype_code(out.dtype),
            _stream(stream)))
        return out

    def window_decode_step(self, keys, values, block_tables, start_pos, seq_lens, max_seq_len: int,
                           q, window: int, sinks: int = 0, scale: float = 1.0, out=None,
                           dtype=torch.bfloat16, stream=None):
        """append(keys, values, ...) of one token per sequence at start_pos
        (= seq_lens - 1), then window_attention, in one call. keys/values bf16
        [n_seqs, 1, n_kv_heads, D]."""
        n, heads, _ = _check_tensor("q", q, torch.bfloat16, (None, None, self._D))
        _check_tensor("keys", keys, torch.bfloat16, (n, 1, self._H, self._D))
        _check_tensor("values", values, torch.bfloat16, (n, 1, self._H, self._D))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        _check_tensor("start_pos", start_pos, torch.int32, (n,))
        _check_tensor("seq_lens", seq_lens, torch.int32, (n,))
        _check_window(window, sinks, max_seq_len)
        dev = self._device
        out = _out(out, q, dtype, stream)
        _check(self._lib.fmkv_paged_window_decode_step(
            self._h, _here(keys, dev), _here(values, dev), _here(block_tables, dev), width,
            _here(start_pos, dev), _here(seq_lens, dev), n, max_seq_len, _here(q, dev), heads,
            scale, window, sinks, _here(out, dev), _dtype_code(out.dtype), _stream(stream)))
        return out

    def window_prefill(self, q, block_tables, start_pos, window: int, sinks: int = 0,
                       scale: float = 1.0, max_seq_len: int = 0, out=None, dtype=torch.bfloat16,
                       stream=None):
        """Attention of q bf16 [n_seqs, n_new, n_q_heads, D] at positions
        start_pos .. start_pos + n_new - 1, whose keys and values were appended
        before, over the window and the sinks of each. max_seq_len: see
        prefill_step."""
        n, n_new, heads, _ = _check_tensor("q", q, torch.bfloat16, (None, None, None, self._D))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        _check_tensor("start_pos", start_pos, torch.int32, (n,))
        _check_window(window, sinks, max_seq_len)
        dev = self._device
        out = _out(out, q, dtype, stream)
        _check(self._lib.fmkv_paged_window_prefill_attention(
            self._h, _here(q, dev), _here(block_tables, dev), width, _here(start_pos, dev), n,
            n_new, max_seq_len, heads, scale, window, sinks, _here(out, dev),
            _dtype_code(out.dtype), _stream(stream)))
        return out

    def window_prefill_step(self, keys, values, block_tables, start_pos, q, window: int,
                            sinks: int = 0, scale: float = 1.0, max_seq_len: int = 0, out=None,
                            dtype=torch.bfloat16, stream=None):
        """append(keys, values, ...) at start_pos, then window_prefill(q, ...).
        keys/values bf16 [n_seqs, n_new, n_kv_heads, D]."""
        n, n_new, heads, _ = _check_tensor("q", q, torch.bfloat16, (None, None, None, self._D))
        _check_tensor("keys", keys, torch.bfloat16, (n, n_new, self._H, self._D))
        _check_tensor("values", values, torch.bfloat16, (n, n_new, self._H, self._D))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        _check_tensor("start_pos", start_pos, torch.int32, (n,))
        _check_window(window, sinks, max_seq_len)
        dev = self._device
        out = _out(out, q, dtype, stream)
        _check(self._lib.fmkv_paged_window_prefill_step(
            self._h, _here(keys, dev), _here(values, dev), _here(block_tables, dev), width,
            _here(start_pos, dev), n, n_new, max_seq_len, _here(q, dev), heads, scale, window, sinks,
            _here(out, dev), _dtype_code(out.dtype), _stream(stream)))
        return out

    def prefix_attention(self, q, block_tables, seq_lens, prefix_lens, group_starts,
                         max_prefix_len: int, max_rest_len: int, scale: float = 1.0, out=None,
                         dtype=torch.bfloat16, stream=None):
        """attention() of a batch in groups that share prefixes, each prefix read
        once for its group: the sequences group_starts[g] .. group_starts[g + 1] - 1
        have the whole blocks of their first prefix_lens[s] positions in common. q bf16
        [n_seqs, n_q_heads, D]; seq_lens, prefix_lens int32 [n_seqs]; group_starts
        int32 [n_groups + 1]. max_prefix_len bounds the prefixes, max_rest_len what a
        sequence holds behind its shared blocks."""
        n, heads, _ = _check_tensor("q", q, torch.bfloat16, (None, None, self._D))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        _check_tensor("seq_lens", seq_lens, torch.int32, (n,))
        groups = _check_groups(prefix_lens, group_starts, n, max_prefix_len, max_rest_len)
        dev = self._device
        out = _out(out, q, dtype, stream)
        _check(self._lib.fmkv_paged_prefix_decode_attention(
            self._h, _here(q, dev), _here(block_tables, dev), width, _here(seq_lens, dev), n,
            _here(prefix_lens, dev), _here(group_starts, dev), groups, max_prefix_len, max_rest_len,
            heads, scale, _here(out, dev), _dtype_code(out.dtype), _stream(stream)))
        return out

    def prefix_decode_step(self, keys, values, block_tables, start_pos, seq_lens, prefix_lens,
                           group_starts, max_prefix_len: int, max_rest_len: int, q,
                           scale: float = 1.0, out=None, dtype=torch.bfloat16, stream=None):
        """append(keys, values, ...) of one token per sequence at start_pos
        (= seq_lens - 1, behind the shared blocks), then prefix_attention, in one
        call. keys/values bf16 [n_seqs, 1, n_kv_heads, D]."""
        n, heads, _ = _check_tensor("q", q, torch.bfloat16, (None, None, self._D))
        _check_tensor("keys", keys, torch.bfloat16, (n, 1, self._H, self._D))
        _check_tensor("values", values, torch.bfloat16, (n, 1, self._H, self._D))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        _check_tensor("start_pos", start_pos, torch.int32, (n,))
        _check_tensor("seq_lens", seq_lens, torch.int32, (n,))
        groups = _check_groups(prefix_lens, group_starts, n, max_prefix_len, max_rest_len)
        dev = self._device
        out = _out(out, q, dtype, stream)
        _check(self._lib.fmkv_paged_prefix_decode_step(
            self._h, _here(keys, dev), _here(values, dev), _here(block_tables, dev), width,
            _here(start_pos, dev), _here(seq_lens, dev), n, _here(prefix_lens, dev),
            _here(group_starts, dev), groups, max_prefix_len, max_rest_len, _here(q, dev), heads, scale,
            _here(out, dev), _dtype_code(out.dtype), _stream(stream)))
        return out

    def weighing_attention(self, q, block_tables, seq_lens, max_seq_len: int, weights=None,
                           weights_out=None, scale: float = 1.0, out=None, dtype=torch.bfloat16,
                           stream=None):
        """(attention(), accumulated weights): each position's softmax weights,
        summed over the query heads, added to `weights` (None: zeros), f32 [n_seqs,
        at least max_seq_len]. weights_out: a buffer of that shape for the sums (None:
        weights itself, or a new one of max_seq_len); its entries from seq_lens[s]
        on stay as they were (0 in a new one)."""
        n, heads, _ = _check_tensor("q", q, torch.bfloat16, (None, None, self._D))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        _check_tensor("seq_lens", seq_lens, torch.int32, (n,))
        dev = self._device
        weights_out = _sums(weights, weights_out, n, max_seq_len, q, stream)
        out = _out(out, q, dtype, stream)
        _check(self._lib.fmkv_paged_weighing_decode_attention(
            self._h, _here(q, dev), _here(block_tables, dev), width, _here(seq_lens, dev), n,
            max_seq_len, _here(weights, dev), _here(weights_out, dev), weights_out.shape[1], heads,
            scale, _here(out, dev), _dtype_code(out.dtype), _stream(stream)))
        return out, weights_out

    def weighing_decode_step(self, keys, values, block_tables, start_pos, seq_lens,
                             max_seq_len: int, q, weights=None, weights_out=None,
                             scale: float = 1.0, out=None, dtype=torch.bfloat16, stream=None):
        """append(keys, values, ...) of one token per sequence at start_pos
        (= seq_lens - 1), then weighing_attention, in one call. keys/values bf16
        [n_seqs, 1, n_kv_heads, D]."""
        n, heads, _ = _check_tensor("q", q, torch.bfloat16, (None, None, self._D))
        _check_tensor("keys", keys, torch.bfloat16, (n, 1, self._H, self._D))
        _check_tensor("values", values, torch.bfloat16, (n, 1, self._H, self._D))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        _check_tensor("start_pos", start_pos, torch.int32, (n,))
        _check_tensor("seq_lens", seq_lens, torch.int32, (n,))
        dev = self._device
        weights_out = _sums(weights, weights_out, n, max_seq_len, q, stream)
        out = _out(out, q, dtype, stream)
        _check(self._lib.fmkv_paged_weighing_decode_step(
            self._h, _here(keys, dev), _here(values, dev), _here(block_tables, dev), width,
            _here(start_pos, dev), _here(seq_lens, dev), n, max_seq_len, _here(q, dev),
            _here(weights, dev), _here(weights_out, dev), weights_out.shape[1], heads, scale,
            _here(out, dev), _dtype_code(out.dtype), _stream(stream)))
        return out, weights_out

    def attention_weights(self, q, block_tables, start_pos, max_seq_len: int, weights=None,
                          weights_out=None, scale: float = 1.0, stream=None):
        """The accumulated weights alone, of q bf16 [n_seqs, n_new, n_q_heads, D] at
        positions start_pos .. start_pos + n_new - 1, whose keys were appended
        before, each over the positions up to its own; max_seq_len bounds start_pos + n_new.
        weights, weights_out: see weighing_attention. Returns weights_out."""
        n, n_new, heads, _ = _check_tensor("q", q, torch.bfloat16, (None, None, None, self._D))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        _check_tensor("start_pos", start_pos, torch.int32, (n,))
        dev = self._device
        weights_out = _sums(weights, weights_out, n, max_seq_len, q, stream)
        _check(self._lib.fmkv_paged_attention_weights(
            self._h, _here(q, dev), _here(block_tables, dev), width, _here(start_pos, dev), n, n_new,
            max_seq_len, _here(weights, dev), _here(weights_out, dev), weights_out.shape[1], heads,
            scale, _stream(stream)))
        return weights_out

    def compact(self, block_tables, keep, n_keep, dst_tables, stream=None) -> None:
        """Moves the tokens that sequences keep to the front of other blocks:
        position keep[s, i] becomes position i of dst_tables' row s, i <
        n_keep[s]. int32: block_tables [n_seqs, max_blocks], keep [n_seqs,
        max_keep], n_keep [n_seqs], dst_tables [n_seqs, dst_max_blocks]. No
        block of dst_tables is one of a sequence's sources, or listed twice."""
        n, most = _check_tensor("keep", keep, torch.int32, (None, None))
        width = _check_tensor("block_tables", block_tables, torch.int32, (n, None))[1]
        dst_width = _check_tensor("dst_tables", dst_tables, torch.int32, (n, None))[1]
        _check_tensor("n_keep", n_keep, torch.int32, (n,))
        dev = self._device
        _check(self._lib.fmkv_paged_compact(
            self._h, _here(block_tables, dev), width, _here(keep, dev), most, _here(n_keep, dev),
            _here(dst_tables, dev), dst_width, n, _stream(stream)))

    def storage(self) -> torch.Tensor:
        """The pool's blocks as a uint8 tensor [n_blocks, n_kv_heads, bytes of a
        head-block] over the pool's own memory (which it keeps alive, unless
        close() ends it): to move blocks to other pools of the same description
        or to the host and back."""
        base, size = ctypes.c_void_p(), ctypes.c_int64()
        _check(self._lib.fmkv_pool_storage(self._h, ctypes.byref(base), ctypes.byref(size)))
        return torch.as_tensor(_Storage(self, base.value, (
            self.n_blocks, self.desc.n_kv_heads, size.value // self.desc.n_kv_heads)),
            device=f"cuda:{self._device}")

    def read_codes(self, stream=None):
        return _read_codes(self._lib.fmkv_pool_read_codes, self._h, self.desc,
                           self.n_blocks * BLOCK_TOKENS, stream)


def copy_blocks(pools, src, dst, stream=None) -> None:
    """Blocks src[i] to dst[i] in every pool of `pools` (a model's layers), in
    one launch. src, dst: int32 [n] on the device; the destinations are distinct
    and no sources."""
    pools = list(pools)
    _check_tensor("src", src, torch.int32, (None,))
    _check_tensor("dst", dst, torch.int32, (src.shape[0],))
    dev = torch.cuda.current_device()
    handles = (ctypes.c_void_p * max(len(pools), 1))(*[p._h for p in pools])
    _check(load_library().fmkv_pools_copy_blocks(handles, len(pools), _here(src, dev),
                                                 _here(dst, dev), src.shape[0], _stream(stream)))


def heaviest_tokens(weights, seq_lens, max_keep: int, sinks: int = 0, recent: int = 0, keep=None,
                    n_keep=None, weights_out=None, stream=None):
    """(keep, n_keep, weights_out): the positions that each sequence keeps, in
    order, as PagedPool.compact takes them. Of more than max_keep the first `sinks`
    and the last `recent` ones and the heaviest of the others by `weights` (f32
    [n_seqs, width]; equal ones: the lower position); of at most max_keep all.
    weights_out f32 [n_seqs, at least max_keep]: their weights, 0 behind them. keep
    int32 [n_seqs, max_keep] stays as it was behind n_keep[s] (0 in a new one)."""
    n, width = _check_tensor("weights", weights, torch.float32, (None, None))
    _check_tensor("seq_lens", seq_lens, torch.int32, (n,))
    for name, value in (("max_keep", max_keep), ("sinks", sinks), ("recent", recent),
                        ("the width of weights", width)):
        _check_bits(name, value, 32)
    if not 1 <= max_keep <= 2 ** 28 - 16:
        raise ValueError("max_keep must be in [1, 2^28 - 16]")
    dev = torch.cuda.current_device()
    _here(weights, dev)
    with _on(stream):
        if keep is None:
            keep = torch.zeros((n, max_keep), dtype=torch.int32, device=weights.device)
        if n_keep is None:
            n_keep = torch.empty(n, dtype=torch.int32, device=weights.device)
        if weights_out is None:
            weights_out = torch.empty((n, max_keep), dtype=torch.float32, device=weights.device)
    _check_tensor("keep", keep, torch.int32, (n, max_keep))
    _check_tensor("n_keep", n_keep, torch.int32, (n,))
    kept_width = _check_tensor("weights_out", weights_out, torch.float32, (n, None))[1]
    _check_bits("the width of weights_out", kept_width, 32)
    _check(load_library().fmkv_heaviest_tokens(
        _here(weights, dev), width, _here(seq_lens, dev), n, max_keep, sinks, recent,
        _here(keep, dev), _here(n_keep, dev), _here(weights_out, dev), kept_width, _stream(stream)))
    return keep, n_keep, weights_out


def qkv_norm_rope(q, k, v, positions, prologue: QkvPrologue, out=None, stream=None):
    """(q, k, v) of a layer from its projections in one pass: per-head norms of
    all three, q and k rotated by their positions (src/model/gemma4_attention.rs
    :50-81). q bf16 [n_tokens, n_q_heads, D], k and v [n_tokens, n_kv_heads, D],
    each row of heads contiguous and tokens any stride apart (slices of a fused
    projection); q, or k and v, may be None. positions int32 [n_axes, n_tokens]
    ([n_tokens] with one axis). Returns contiguous rows for append, decode_step
    and the prefill calls (None for what was not given; with v_from_k V comes
    from k). out: the three outputs, which may be the inputs themselves."""
    if q is None and k is None:
        raise ValueError("q or k must be given")
    dev = torch.cuda.current_device()
    n, _, D = (k if q is None else q).shape
    for w in getattr(prologue, "weights", ()):
        if w is None:
            continue
        if w.shape[0] != D:
            raise ValueError(f"a norm weight has {w.shape[0]} elements; head_dim is {D}")
        if w.get_device() != dev:
            raise ValueError(f"a norm weight is on {w.device}, not on the current GPU")
    q_heads, q_ptr, q_stride = _head_rows("q", q, n, D, dev)
    k_heads, k_ptr, k_stride = _head_rows("k", k, n, D, dev)
    v_heads, v_ptr, v_stride = _head_rows("v", v, n, D, dev)
    if v is not None and v_heads != k_heads:
        raise ValueError("v needs a k of its shape")
    if positions is not None:
        axes = prologue.n_axes
        _check_tensor("positions", positions, torch.int32,
                      (n,) if axes == 1 and positions.dim() == 1 else (axes, n))
    like = (q, k, k if prologue.v_from_k else v)
    if out is None:
        with _on(stream):
            out = tuple(None if t is None else
                        torch.empty_like(t, memory_format=torch.contiguous_format) for t in like)
    else:
        for t, o in zip(like, out):
            if (t is None) != (o is None):
                raise ValueError("out must have a tensor for each output")
            if t is not None:
                _check_tensor("out", o, torch.bfloat16, tuple(t.shape))
        out = tuple(out)
    if n == 0:
        return out
    _check(load_library().fmkv_qkv_norm_rope(
        ctypes.byref(prologue), D, q_heads, k_heads, n, q_ptr, q_stride, k_ptr, k_stride, v_ptr,
        v_stride, _here(positions, dev), _here(out[0], dev), _here(out[1], dev), _here(out[2], dev),
        _stream(stream)))
    return out


def _head_rows(name: str, t, n: int, D: int, dev: int):
    """(heads, address, elements from token to token) of rows [n, heads, D]."""
    if t is None:
        return 0, None, 0
    heads = _check_tensor(name, t, torch.bfloat16, (n, None, D))[1]
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s1 != D and heads > 1) or t.get_device() != dev:
        raise ValueError(f"{name} must be on the current GPU, with contiguous rows of heads")
    return heads, t.data_ptr(), s0 if n > 1 else heads * D


class PageBook:
    """The book of a pool's blocks (or of several pools that share their block
    tables): which are free, how many sequences use each. Block lists are host
    lists of ints (-1: given back)."""

    def __init__(self, n_blocks: int):
        _check_bits("n_blocks", n_blocks, 64)
        self.n_blocks = n_blocks
        self._lib = load_library()
        h = ctypes.c_void_p()
        _check(self._lib.fmkv_pages_create(n_blocks, ctypes.byref(h)))
        self._h = h

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.fmkv_pages_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def free_count(self) -> int:
        v = ctypes.c_int64()
        _check(self._lib.fmkv_pages_free_count(self._h, ctypes.byref(v)))
        return v.value

    def users(self, block: int) -> int:
        v = ctypes.c_int32()
        _check(self._lib.fmkv_pages_users(self._h, _i32s([block])[0], ctypes.byref(v)))
        return v.value

    def alloc(self, n: int) -> list[int]:
        """n free blocks (an error, and none taken, when fewer are free)."""
        _check_bits("n", n, 64)
        if n > self.n_blocks:
            raise Exception_(FMKV_ERR_CAPACITY, f"{n} blocks asked for of {self.n_blocks}")
        buf = (ctypes.c_int32 * max(n, 1))()
        _check(self._lib.fmkv_pages_alloc(self._h, n, buf))
        return list(buf[:max(n, 0)])

    def release(self, blocks) -> None:
        """One user less for each block."""
        blocks = list(blocks)
        _check(self._lib.fmkv_pages_release(self._h, _i32s(blocks), len(blocks)))

    def fork(self, blocks, n_tokens: int):
        """(blocks of a second sequence that goes on from n_tokens of a first,
        the (src, dst) copy that copy_blocks has to make for it or None)."""
        _check_bits("n_tokens", n_tokens, 64)
        blocks = list(blocks)
        n = (n_tokens + BLOCK_TOKENS - 1) // BLOCK_TOKENS
        if n > len(blocks):
            raise ValueError(f"{n_tokens} tokens need {n} blocks, got {len(blocks)}")
        child, src, dst = (ctypes.c_int32 * max(n, 1))(), ctypes.c_int32(), ctypes.c_int32()
        _check(self._lib.fmkv_pages_fork(self._h, _i32s(blocks), n_tokens, child, ctypes.byref(src),
                                         ctypes.byref(dst)))
        return list(child[:max(n, 0)]), None if src.value < 0 else (src.value, dst.value)

    def slide(self, blocks, n_tokens: int, window: int, sinks: int = 0) -> list[int]:
        """The sequence's blocks after giving back those that no query at position
        n_tokens or later sees through the window and the sinks (-1 there)."""
        _check_bits("n_tokens", n_tokens, 64)
        blocks = list(blocks)
        if (n_tokens + BLOCK_TOKENS - 1) // BLOCK_TOKENS > len(blocks):
            raise ValueError(f"{n_tokens} tokens need more than {len(blocks)} blocks")
        _check_window(window, sinks)
        buf, n = _i32s(blocks), ctypes.c_int64()
        _check(self._lib.fmkv_pages_slide(self._h, buf, n_tokens, window, sinks, ctypes.byref(n)))
        return list(buf[:len(blocks)])


def _check_bits(name: str, value: int, bits: int) -> None:
    """ctypes passes on the low bits of a number that is too wide for the
    argument, another number, which the library cannot tell from a good one."""
    if not -(1 << bits - 1) <= value < 1 << bits - 1:
        raise ValueError(f"{name} does not fit {bits} bits")


def _i32s(values):
    # (ctypes would keep the low 32 bits of a larger number, another block's)
    if values and (min(values) < -2 ** 31 or max(values) >= 2 ** 31):
        raise ValueError("a block does not fit 32 bits")
    return (ctypes.c_int32 * max(len(values), 1))(*values)


class _Storage:
    """A pool's memory for torch (the tensor holds this object, and it the pool)."""

    def __init__(self, owner, ptr: int, shape):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": tuple(shape),
                                         "typestr": "|u1", "strides": None, "version": 2}


def _check_window(window: int, sinks: int, max_seq_len: int = 0) -> None:
    """Values whose low 32 bits ctypes would pass on (the library checks the rest)."""
    if not (-2 ** 31 <= window < 2 ** 31 and -2 ** 31 <= sinks < 2 ** 31):
        raise ValueError("window and sinks must be at most 2^30")
    _check_bits("max_seq_len", max_seq_len, 32)


def _check_groups(prefix_lens, group_starts, n: int, max_prefix_len: int, max_rest_len: int) -> int:
    """Number of groups of a batch that shares prefixes."""
    _check_tensor("prefix_lens", prefix_lens, torch.int32, (n,))
    ends = _check_tensor("group_starts", group_starts, torch.int32, (None,))[0]
    if ends < 1:
        raise ValueError("group_starts must have n_groups + 1 entries")
    _check_bits("max_prefix_len", max_prefix_len, 32)
    _check_bits("max_rest_len", max_rest_len, 32)
    return ends - 1


def _sums(weights, weights_out, n: int, max_seq_len: int, like: torch.Tensor, stream):
    """Where accumulated weights go: weights_out, weights itself, or a new buffer."""
    _check_bits("max_seq_len", max_seq_len, 32)
    if weights is not None:
        width = _check_tensor("weights", weights, torch.float32, (n, None))[1]
        if weights_out is None:
            weights_out = weights
        _check_tensor("weights_out", weights_out, torch.float32, (n, width))
    elif weights_out is None:
        with _on(stream):
            weights_out = torch.zeros((n, max(max_seq_len, 1)), dtype=torch.float32, device=like.device)
    _check_bits("the width of weights_out", _check_tensor("weights_out", weights_out, torch.float32,
                                                          (n, None))[1], 32)
    return weights_out


def _check_tensor(name: str, t: torch.Tensor, dtype, shape):
    """Type and shape (None: any extent) of an argument that the library takes as
    a bare pointer; its shape."""
    have = t.shape
    if t.dtype is dtype and len(have) == len(shape):
        for n, want in zip(have, shape):
            if n != want and want is not None:
                break
        else:
            return have
    want = ", ".join("*" if x is None else str(x) for x in shape)
    raise ValueError(f"{name} must be {dtype} [{want}], got {t.dtype} {tuple(have)}")


def _out(out, like: torch.Tensor, dtype, stream) -> torch.Tensor:
    if out is None:
        if stream is None:
            return torch.empty_like(like, dtype=dtype)
        with _on(stream):
            return torch.empty_like(like, dtype=dtype)
    if out.shape != like.shape:
        raise ValueError(f"out must have the shape {tuple(like.shape)}, got {tuple(out.shape)}")
    return out


def _dtype_code(dtype) -> int:
    if dtype == torch.bfloat16:
        return DTYPE_BF16
    if dtype == torch.float32:
        return DTYPE_F32
    raise ValueError(f"unsupported output dtype {dtype}")


def words_per_row(desc: CacheDesc) -> int:
    return (desc.head_dim * desc.bits + 31) // 32


def meta_per_row(desc: CacheDesc) -> int:
    if desc.mode == MODE_PLAIN:
        return 0
    return 2 * (desc.head_dim // 64) if desc.mode == MODE_AFFINE else 1


def _read_codes(fn, handle, desc, n_slots, stream):
    H = desc.n_kv_heads
    codes = torch.zeros((n_slots, 2, H, words_per_row(desc)), dtype=torch.int32, device="cuda")
    meta = torch.zeros((n_slots, 2, H, meta_per_row(desc)), dtype=torch.int16, device="cuda")
    _check(fn(handle, _ptr(codes), _ptr(meta), _stream(stream)))
    return codes, meta
