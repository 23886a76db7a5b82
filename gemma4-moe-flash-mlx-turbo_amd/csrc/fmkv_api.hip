// C ABI of the MI355X quantized KV cache (include/fmkv.h).
//
// Host-side state mirrors KVCache (src/cache.rs:166-172): the monotonic
// `offset` (RoPE position), the optional sliding `window`, and the stored
// K/V -- here a preallocated device arena of 16-token head-blocks instead of
// MLX arrays re-concatenated on every append (src/cache.rs:132-148).
// Errors never cross the boundary as exceptions: every entry point returns a
// status and records a message for fmkv_last_error().
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <exception>
#include <mutex>
#include <string>
#include <utility>
#include <vector>

#include "../../include/fmkv.h"
#include "fmkv_internal.h"

using fmkv::BlockLayout;

namespace {

thread_local std::string g_err;
int32_t g_bps_override = 0;
// sparse-V after the statistics pass: 1 the gather, 0 the gated pass and the
// combine (fmkv_set_sparse_v_gather)
int32_t g_sparse_gather = 1;

// Kernel-timing records (fmkv_profile_enable / fmkv_profile_collect).
struct Profiler {
  std::vector<hipEvent_t> ev;  // pairs
  int32_t max_records = 0;
  int32_t used = 0;
  void clear_events() {
    for (hipEvent_t e : ev) (void)hipEventDestroy(e);
    ev.clear();
    used = 0;
  }
} g_prof;

// Next event pair for a decode launch, or {null, null} when not profiling.
void next_events(hipEvent_t* e0, hipEvent_t* e1) {
  *e0 = *e1 = nullptr;
  if (g_prof.max_records <= 0 || g_prof.used >= g_prof.max_records) return;
  const size_t i = 2 * (size_t)g_prof.used;
  *e0 = g_prof.ev[i];
  *e1 = g_prof.ev[i + 1];
  g_prof.used++;
}

int fail(int code, const std::string& msg) {
  g_err = msg;
  return code;
}

int hip_fail(hipError_t e, const char* what) {
  return fail(FMKV_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

// src/cache.rs:29-43: MMIX LCG stepped before each draw, +1 iff bit 63 == 0.
std::vector<float> lcg_signs(int n, uint64_t seed) {
  std::vector<float> s(n);
  uint64_t state = seed;
  for (int i = 0; i < n; i++) {
    state = state * 6364136223846793005ull + 1442695040888963407ull;
    s[i] = ((state >> 63) & 1ull) == 0 ? 1.0f : -1.0f;
  }
  return s;
}

int check_desc(const fmkv_cache_desc* d) {
  if (!d) return fail(FMKV_ERR_INVALID_ARG, "descriptor is null");
  if (d->n_kv_heads < 1 || d->n_kv_heads > 256)
    return fail(FMKV_ERR_INVALID_ARG, "n_kv_heads must be in [1, 256]");
  if (d->head_dim != 128 && d->head_dim != 256 && d->head_dim != 512)
    return fail(FMKV_ERR_UNSUPPORTED, "head_dim must be 128, 256 or 512");
  if (d->group_size != 64) return fail(FMKV_ERR_UNSUPPORTED, "group_size must be 64");
  if (d->mode == FMKV_MODE_AFFINE) {
    if (d->bits != 4 && d->bits != 8)
      return fail(FMKV_ERR_UNSUPPORTED, "affine mode supports 4 or 8 bits");
  } else if (d->mode == FMKV_MODE_CODEBOOK) {
    if (d->bits < 2 || d->bits > 4)
      return fail(FMKV_ERR_UNSUPPORTED, "codebook mode supports 2, 3 or 4 bits");
  } else if (d->mode == FMKV_MODE_PLAIN) {
    if (d->bits != 16) return fail(FMKV_ERR_UNSUPPORTED, "plain (bf16) mode has bits = 16");
  } else {
    return fail(FMKV_ERR_UNSUPPORTED, "unknown mode");
  }
  if (d->window < 0) return fail(FMKV_ERR_INVALID_ARG, "window must be >= 0");
  if (d->window > 0) {
    if (d->window > (1 << 30)) return fail(FMKV_ERR_INVALID_ARG, "window must be <= 2^30");
  } else {
    if (d->capacity < 1) return fail(FMKV_ERR_INVALID_ARG, "capacity must be >= 1 for a global cache");
    if (d->capacity > ((int64_t)1 << 31) - 64)
      return fail(FMKV_ERR_INVALID_ARG, "capacity must be < 2^31 - 64");
  }
  return FMKV_OK;
}

// Slots of a ring: the sliding window W rounded up to whole 16-token
// head-blocks. Position p is stored at slot p mod ring_slots, so the ring
// holds the last ring_slots positions; the last W of them are visible
// (visible_begin), the others masked by position.
int64_t ring_slots(const fmkv_cache_desc& d) {
  return d.window > 0 ? fmkv::round_up(d.window, fmkv::kBlockTokens) : 0;
}

int64_t n_slots_of(const fmkv_cache_desc& d) {
  return d.window > 0 ? ring_slots(d) : fmkv::round_up(d.capacity, fmkv::kBlockTokens);
}

int device_cus() {
  static std::atomic<int> known[64];  // by device: the query takes as long as a launch
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  if (dev >= 0 && dev < 64 && (cus = known[dev].load(std::memory_order_relaxed)) > 0) return cus;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    return 256;
  if (dev >= 0 && dev < 64) known[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// Decode work-groups per CU the split plan aims at: the affine and codebook
// kernels' LDS staging fills a CU; the plain kernel's work-groups are about
// half as large (two per CU).
int attn_wg_per_cu(const fmkv_cache_desc& d) {
  return d.mode == FMKV_MODE_PLAIN ? 2 : fmkv::kAttnWgPerCu;
}

// Work-groups per CU of a paged batch's decode kernel when its splits are
// long enough for single-wave streams (at least 8 blocks each): 3 for
// affine head-blocks of at most 1024 code bits per token (four-wave
// work-groups), else 1.
int paged_solo_slots(const fmkv_cache_desc& d) {
  return d.mode == FMKV_MODE_AFFINE && d.head_dim * d.bits <= 1024 ? 3 : 1;
}

// Split-K plan: blocks per split such that the grid has about `wg_per_cu`
// work-groups per CU (each keeps several blocks in flight, so one per CU
// already saturates HBM; more would only add split partials), `reserved` of
// them going to other work of the same launch (the new-token column).
int32_t choose_bps(int64_t total_head_blocks, int cus, int wg_per_cu, int64_t reserved = 0,
                   int64_t min_bps = 1) {
  if (g_bps_override > 0) return g_bps_override;
  int64_t target = (int64_t)wg_per_cu * cus;
  if (target - reserved >= target / 2) target -= reserved;
  int64_t bps = (total_head_blocks + target - 1) / target;
  if (bps < min_bps) bps = min_bps;
  if (bps < 1) bps = 1;
  return (int32_t)bps;
}

// src/cache.rs:29-43 signs as a bit mask (bit d set = -1), the form the
// decode kernel takes them in as a kernel argument.
void sign_bits_of(const fmkv_cache_desc& d, uint32_t out[16]) {
  std::vector<float> s = lcg_signs(d.head_dim, d.sign_seed);
  for (int w = 0; w < 16; w++) out[w] = 0;
  for (int i = 0; i < d.head_dim; i++)
    if (s[i] < 0.0f) out[i >> 5] |= 1u << (i & 31);
}

// Caller-provided device memory standing in for a handle's workspace (the
// no-allocation decode step); ptr null: the handle's own workspace.
struct ExtWorkspace {
  float* ptr = nullptr;
  size_t bytes = 0;
};

// The call on stream s becomes part of a graph.
bool is_captured(hipStream_t s) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  const bool captured = hipStreamIsCapturing(s, &st) != hipSuccess || st != hipStreamCaptureStatusNone;
  if (captured) (void)hipGetLastError();
  return captured;
}

// Allocating does not end a capture in a thread's relaxed mode.
struct RelaxedCapture {
  hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
  RelaxedCapture() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
  ~RelaxedCapture() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
};

struct Workspace {
  float* ptr = nullptr;
  size_t bytes = 0;
  // A pool's calls say whether they are captured. What a captured call uses stays
  // until the handle's end, since its graph uses it at every replay; an outgrown
  // buffer of eager calls alone is freed.
  bool captured = false;  // the call being prepared
  bool in_graph = false;  // ptr: an earlier one
  std::vector<float*> kept;
  // zero: a new allocation starts zeroed (head-block staging, whose
  // unwritten slots are read, masked, as the cache's own are)
  int ensure(size_t need, bool zero = false) {
    if (need > bytes) {
      const int rc = captured || in_graph ? grow(need) : replace(need, zero);
      if (rc) return rc;
    }
    in_graph = in_graph || captured;
    return FMKV_OK;
  }
  int replace(size_t need, bool zero) {
    if (ptr) (void)hipFree(ptr);  // (waits for the calls that use it)
    ptr = nullptr;
    bytes = 0;
    hipError_t e = hipMalloc(&ptr, need);
    if (e != hipSuccess) {
      ptr = nullptr;
      (void)hipGetLastError();
      return fail(FMKV_ERR_OOM, "workspace allocation failed");
    }
    if (zero) {
      e = hipMemset(ptr, 0, need);
      if (e != hipSuccess) return hip_fail(e, "hipMemset(workspace)");
    }
    bytes = need;
    return FMKV_OK;
  }
  // Half as large again where memory allows, so that the buffers kept together
  // stay below twice the last; else what the call needs.
  int grow(size_t need) {
    size_t want = std::max(need, bytes + bytes / 2);
    try {
      kept.reserve(kept.size() + 1);
    } catch (const std::exception&) {
      return fail(FMKV_ERR_OOM, "no host memory for a workspace");
    }
    float* p = nullptr;
    hipError_t e = hipMalloc(&p, want);
    if (e != hipSuccess && want > need) {
      (void)hipGetLastError();
      want = need;
      e = hipMalloc(&p, want);
    }
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return fail(FMKV_ERR_OOM, "workspace allocation failed");
    }
    if (ptr) kept.push_back(ptr);
    ptr = p;
    bytes = want;
    in_graph = false;
    return FMKV_OK;
  }
  void release() {
    for (float* p : kept) (void)hipFree(p);
    kept.clear();
    if (ptr) (void)hipFree(ptr);
    ptr = nullptr;
    bytes = 0;
  }
};

constexpr int kMaxDevices = 64;

// The partials of split prefill calls: one buffer per GPU for all its handles
// (a call's partials live only while it runs, and a split grid fills the chip,
// so two would not run side by side anyway). The first split call allocates it,
// at the size that any call may need, and the last handle of the GPU frees it.
// Calls on several streams and from several threads (of different handles) may
// be in flight, so each use waits, on its stream, for the one before; the lock
// keeps a use's wait, launches and record together.
struct PrefillScratch {
  std::mutex mu;
  int handles = 0;
  float* ptr = nullptr;
  size_t bytes = 0;
  hipEvent_t used = nullptr;

  // The buffer is there (false: no memory for it). Not a reason for a capture
  // on another stream or thread to fail: allocating is allowed in this
  // thread's relaxed mode.
  bool ready(int cus) {
    if (ptr) return true;
    RelaxedCapture relaxed;
    bytes = fmkv::prefill_scratch_bytes(cus);
    if (hipMalloc(&ptr, bytes) != hipSuccess) ptr = nullptr;
    if (ptr && hipEventCreateWithFlags(&used, hipEventDisableTiming) != hipSuccess) {
      (void)hipFree(ptr);
      ptr = nullptr;
    }
    if (!ptr) (void)hipGetLastError();
    return ptr != nullptr;
  }
};
PrefillScratch g_prefill_scratch[kMaxDevices];

// A handle's part in its GPU's scratch, from its creation to its end.
PrefillScratch* prefill_scratch_join() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return nullptr;
  PrefillScratch* sc = &g_prefill_scratch[dev];
  std::lock_guard<std::mutex> lock(sc->mu);
  sc->handles++;
  return sc;
}
void prefill_scratch_leave(PrefillScratch* sc) {
  if (!sc) return;
  std::lock_guard<std::mutex> lock(sc->mu);
  if (--sc->handles > 0 || !sc->ptr) return;
  (void)hipFree(sc->ptr);  // (waits for the calls that use it)
  (void)hipEventDestroy(sc->used);
  sc->ptr = nullptr;
  sc->used = nullptr;
}

}  // namespace

struct fmkv_cache {
  fmkv_cache_desc desc;
  BlockLayout layout;
  uint8_t* arena;
  int64_t n_blocks;
  float* d_signs;
  uint32_t sign_bits[16];
  float c, sqrt_d;
  int64_t offset;
  int64_t vis_begin;
  Workspace ws;
  Workspace stage;  // prefill on a ring: the chunk's quantized rows
  PrefillScratch* split = nullptr;
  int cus;
};

struct fmkv_pool {
  fmkv_cache_desc desc;
  BlockLayout layout;
  uint8_t* arena;
  int64_t n_blocks;
  float* d_signs;
  uint32_t sign_bits[16];
  float c, sqrt_d;
  Workspace ws;
  PrefillScratch* split = nullptr;
  int cus;
  int device;  // the GPU that holds the pool
};

namespace {

fmkv::Store cache_store(const fmkv_cache* c) {
  fmkv::Store s;
  s.base = c->arena;
  s.block_stride = c->layout.block_bytes;
  s.head_stride = c->n_blocks * c->layout.block_bytes;
  s.block_table = nullptr;
  s.table_stride = 0;
  s.n_blocks = c->n_blocks;
  s.n_kv_heads = c->desc.n_kv_heads;
  s.layout = c->layout;
  return s;
}

fmkv::Store pool_store(const fmkv_pool* p, const int32_t* table, int32_t stride) {
  fmkv::Store s;
  s.base = p->arena;
  s.block_stride = p->layout.block_bytes * p->desc.n_kv_heads;
  s.head_stride = p->layout.block_bytes;
  s.block_table = table;
  s.table_stride = stride;
  s.n_blocks = p->n_blocks;
  s.n_kv_heads = p->desc.n_kv_heads;
  s.layout = p->layout;
  return s;
}

constexpr size_t kOwnPartials = (size_t)8 << 20;

// The prefill attention, split over its keys when the grid alone would leave
// CUs idle. Not under stream capture (a replay would not be ordered with other
// uses of the partials) and not when there is no memory for the partials: the
// unsplit launch needs none. A call that has a workspace of its own (own: a
// windowed call's pool, whose uses the caller orders) is split there where it is
// captured, or its partials are so few that every pool may hold them: 5
// queries after 3000 positions, 8/4 heads of 128 dims, bf16, in a graph 16.3 us,
// unsplit 50.5; eager 17.4, with the shared buffer's wait and event 20.2.
hipError_t run_prefill(fmkv::PrefillArgs& pa, PrefillScratch* sc, int cus, int64_t max_steps,
                       hipStream_t s, Workspace* own = nullptr) {
  const bool captured = is_captured(s);
  // (bytes = rows * (D + 2) floats)
  auto place = [&](float* p, size_t bytes) {
    const int D = pa.new_st.layout.head_dim;
    pa.part_o = p;
    pa.part_ml = p + bytes / sizeof(float) / (D + 2) * D;
  };
  const size_t bytes = fmkv::prefill_plan(pa, cus, max_steps, own || (sc && !captured));
  if (own && bytes > 0 && (captured || !sc || bytes <= kOwnPartials)) {
    RelaxedCapture relaxed;
    own->captured = captured;
    if (own->ensure(bytes) == FMKV_OK)
      place(own->ptr, bytes);
    else
      (void)fmkv::prefill_plan(pa, cus, max_steps, false);
    return fmkv::launch_prefill_attention(pa, s);
  }
  if (bytes == 0) return fmkv::launch_prefill_attention(pa, s);
  std::lock_guard<std::mutex> lock(sc->mu);
  if (!sc->ready(cus) || bytes > sc->bytes) {
    (void)fmkv::prefill_plan(pa, cus, max_steps, false);
    return fmkv::launch_prefill_attention(pa, s);
  }
  place(sc->ptr, bytes);
  hipError_t e = hipStreamWaitEvent(s, sc->used, 0);
  if (e != hipSuccess) return e;
  e = fmkv::launch_prefill_attention(pa, s);
  if (e != hipSuccess) return e;
  return hipEventRecord(sc->used, s);
}

int64_t visible_begin(const fmkv_cache* c) {
  int64_t b = c->vis_begin;
  if (c->desc.window > 0 && c->offset - c->desc.window > b) b = c->offset - c->desc.window;
  return b < 0 ? 0 : b;
}

int make_signs(const fmkv_cache_desc& d, float** out) {
  std::vector<float> s = lcg_signs(d.head_dim, d.sign_seed);
  hipError_t e = hipMalloc(out, sizeof(float) * d.head_dim);
  if (e != hipSuccess) return fail(FMKV_ERR_OOM, "sign vector allocation failed");
  e = hipMemcpy(*out, s.data(), sizeof(float) * d.head_dim, hipMemcpyHostToDevice);
  if (e != hipSuccess) return hip_fail(e, "hipMemcpy(signs)");
  return FMKV_OK;
}

int check_attn_args(const fmkv_cache_desc& d, const void* q, int32_t n_q_heads, float tau,
                    const void* out, int32_t out_dtype) {
  if (!q || !out) return fail(FMKV_ERR_INVALID_ARG, "q/out must be device pointers");
  if (n_q_heads < d.n_kv_heads || n_q_heads % d.n_kv_heads != 0)
    return fail(FMKV_ERR_INVALID_ARG, "n_q_heads must be a multiple of n_kv_heads");
  if (n_q_heads / d.n_kv_heads > 8)
    return fail(FMKV_ERR_UNSUPPORTED, "at most 8 query heads per KV head");
  if (!(tau >= 0.0f) || !std::isfinite(tau))
    return fail(FMKV_ERR_INVALID_ARG, "sparse_v_tau must be finite and >= 0");
  if (out_dtype != FMKV_DTYPE_BF16 && out_dtype != FMKV_DTYPE_F32)
    return fail(FMKV_ERR_INVALID_ARG, "out_dtype must be FMKV_DTYPE_BF16 or FMKV_DTYPE_F32");
  return FMKV_OK;
}

// Validation and launch arguments of an append of n tokens at the cache's
// offset (no state change).
// The layer prologue's arguments (no HIP call): a k_norm
// weight, positive finite eps and theta, rope_dims a power of 2 in
// [2 * head_dim / 64, head_dim] (the rotated pairs then sit in different
// lanes of the append kernel's row layout).
int check_prologue(const fmkv_cache_desc& d, const fmkv_kv_prologue* pro) {
  if (!pro) return fail(FMKV_ERR_INVALID_ARG, "prologue is null");
  if (!pro->k_norm_weight) return fail(FMKV_ERR_INVALID_ARG, "k_norm_weight must be a device pointer");
  if (!(pro->eps > 0.0f) || !std::isfinite(pro->eps))
    return fail(FMKV_ERR_INVALID_ARG, "eps must be finite and > 0");
  if (!(pro->rope_theta > 0.0f) || !std::isfinite(pro->rope_theta))
    return fail(FMKV_ERR_INVALID_ARG, "rope_theta must be finite and > 0");
  const int rd = pro->rope_dims;
  if (rd < 2 * (d.head_dim / 64) || rd > d.head_dim || (rd & (rd - 1)) != 0)
    return fail(FMKV_ERR_UNSUPPORTED,
                "rope_dims must be a power of 2 in [2 * head_dim / 64, head_dim]");
  if (pro->v_from_k != 0 && pro->v_from_k != 1)
    return fail(FMKV_ERR_INVALID_ARG, "v_from_k must be 0 or 1");
  return FMKV_OK;
}

void set_prologue(const fmkv_kv_prologue* pro, fmkv::AppendArgs* a) {
  a->k_norm_w = static_cast<const uint16_t*>(pro->k_norm_weight);
  a->eps = pro->eps;
  a->rope_dims = pro->rope_dims;
  a->rope_theta = pro->rope_theta;
  a->v_from_k = pro->v_from_k;
}

int prepare_append(const fmkv_cache* c, const void* k, const void* v, int64_t n,
                   fmkv::AppendArgs* a, int64_t* tasks) {
  if (!c) return fail(FMKV_ERR_INVALID_ARG, "cache is null");
  if (n < 0) return fail(FMKV_ERR_INVALID_ARG, "n_tokens must be >= 0");
  if (n == 0) return FMKV_OK;
  if (!k || !v) return fail(FMKV_ERR_INVALID_ARG, "k/v must be device pointers");
  if (n > ((int64_t)1 << 30)) return fail(FMKV_ERR_INVALID_ARG, "n_tokens too large");
  const int64_t W = ring_slots(c->desc);  // ring slots (0: linear)
  if (W == 0 && c->offset + n > c->desc.capacity)
    return fail(FMKV_ERR_CAPACITY, "append of " + std::to_string(n) + " tokens at offset " +
                                       std::to_string(c->offset) + " exceeds capacity " +
                                       std::to_string(c->desc.capacity));
  if (c->offset + n > ((int64_t)1 << 31) - 64)
    return fail(FMKV_ERR_CAPACITY, "position counter would exceed 2^31");
  a->st = cache_store(c);
  a->k = static_cast<const uint16_t*>(k);
  a->v = static_cast<const uint16_t*>(v);
  a->start_pos = nullptr;
  a->start_scalar = c->offset;
  a->n_new = (int32_t)n;
  a->window = (int32_t)W;
  std::memcpy(a->sign_bits, c->sign_bits, sizeof(a->sign_bits));
  a->c = c->c;
  a->sqrt_d = c->sqrt_d;
  a->cb_bits = c->desc.bits;
  if (W > 0) {
    const int64_t n_eff = n < W ? n : W;
    *tasks = (n_eff + fmkv::kBlockTokens - 1) / fmkv::kBlockTokens + 1;
    if (*tasks > W / fmkv::kBlockTokens) *tasks = W / fmkv::kBlockTokens;
  } else {
    *tasks = (c->offset + n - 1) / fmkv::kBlockTokens - c->offset / fmkv::kBlockTokens + 1;
  }
  return FMKV_OK;
}

// Split-K plan of one decode attention launch: blocks per split (bps, bps0
// for split 0), split columns per sequence and the XCD-aware skew.
void plan_splits(int cus, int H, int32_t n_seqs, int64_t nblk, int wg_per_cu, int min_bps,
                 int first_mult, int new_col, bool paged, fmkv::AttnArgs* a) {
  if (nblk < 1) nblk = 1;
  // one sequence: the new-token column takes CUs of its own; many sequences:
  // the dispatcher fills CUs as work-groups finish
  const int64_t reserved = n_seqs == 1 ? (int64_t)new_col * H : 0;
  a->bps = choose_bps(nblk * H * n_seqs, cus, wg_per_cu, reserved, min_bps);
  // the split columns are the grid's z dimension (at most 65535)
  if ((nblk + a->bps - 1) / a->bps + new_col > 65535)
    a->bps = (int32_t)((nblk + 65534 - new_col) / (65535 - new_col));
  // split 0 of each sequence takes first_mult x bps blocks
  const int64_t bps0 = (int64_t)a->bps * first_mult;
  a->bps0 = (int32_t)(bps0 < nblk ? bps0 : nblk);
  if (a->bps0 < a->bps) a->bps0 = a->bps;
  a->max_splits = (int32_t)(nblk <= a->bps0 ? 1 : 1 + (nblk - a->bps0 + a->bps - 1) / a->bps);
  a->skew_p = a->skew_extra = 0;
  // XCD-aware plan for one sequence over two KV heads at one work-group per
  // CU: the work-groups (KV head h, split s) go round-robin to the 8 XCDs by
  // linear id h + 2 s, so the splits s = 0 mod 4 land on XCDs 0 and 1, which
  // start first (the others start 1.4 to 4.4 us later). Every CU gets a split
  // of bps blocks and the blocks left over go one each to the splits
  // s = 0 mod p, p = 4 when they fit there (else 2, else 1: the first
  // splits), instead of bps + 1 blocks for every work-group and some CUs
  // left idle.
  if (n_seqs == 1 && H == 2 && wg_per_cu == 1 && !paged &&
      g_bps_override <= 0) {
    const int64_t n_s = (cus - (int64_t)new_col * H) / H;
    const int64_t b = n_s > 0 ? nblk / n_s : 0;
    const int64_t extra = nblk - n_s * b;
    if (n_s >= 8 && b >= fmkv::kAttnPlanMinSkewBlocks) {
      int p = 4;
      while (p > 1 && extra > (n_s + p - 1) / p) p >>= 1;
      a->bps = a->bps0 = (int32_t)b;
      a->max_splits = (int32_t)n_s;
      a->skew_p = p;
      a->skew_extra = (int32_t)extra;
    }
  }
}

// Split-K plan, workspace ([part_o | part_ml]) and launch arguments of
// decode attention; new_col adds the decode step's new-token column.
template <typename Owner>
int prepare_attention_common(Owner* o, const fmkv::Store& st, int32_t n_seqs, int64_t nblk,
                             int64_t blk_cap, const void* q, int32_t n_q_heads, float scale, float tau, void* out,
                             int32_t out_dtype, int wg_per_cu, int min_bps, int first_mult,
                             int new_col, fmkv::AttnArgs* a, ExtWorkspace ext = {}) {
  int rc = check_attn_args(o->desc, q, n_q_heads, tau, out, out_dtype);
  if (rc) return rc;
  const int H = o->desc.n_kv_heads, D = o->desc.head_dim;
  a->st = st;
  a->group = n_q_heads / H;
  a->n_q_heads = n_q_heads;
  a->q = static_cast<const uint16_t*>(q);
  a->qscale = scale * 1.4426950408889634f;
  std::memcpy(a->sign_bits, o->sign_bits, sizeof(a->sign_bits));
  a->c = o->c;
  a->sqrt_d = o->sqrt_d;
  plan_splits(o->cus, H, n_seqs, nblk, wg_per_cu, min_bps, first_mult, new_col,
              st.block_table != nullptr, a);
  a->new_col = new_col;
  a->part_stride = a->max_splits + new_col;
  // sparse-V (tau > 0) always goes through the split partials and the
  // combine, which normalises by the stats pass's full softmax sum
  a->tau = tau;
  a->direct = a->max_splits == 1 && !new_col && tau == 0.0f;
  a->k_new = a->v_new = nullptr;
  a->out = out;
  a->out_f32 = out_dtype == FMKV_DTYPE_F32;
  const size_t n_rows = a->direct ? 0 : (size_t)n_seqs * a->part_stride * n_q_heads;
  // sparse-V: [theta | M | L] per (sequence, q head), then the stats pass's
  // split (m, l) in a region of their own
  const size_t n_stats = tau > 0.0f ? 3 * (size_t)n_seqs * n_q_heads : 0;
  const size_t n_stat_ml = tau > 0.0f ? 2 * n_rows : 0;
  const size_t stat_off = n_rows * (D + 2) + n_stats;
  // sparse-V block maxima, 16-byte aligned (read as float4)
  const size_t blk_off = (stat_off + n_stat_ml + 3) & ~(size_t)3;
  // (rows sized for the most blocks a sequence can hold, so that the
  // library's workspace does not grow as the context does; a caller's
  // scratch holds the call's blocks only)
  a->blk_stride = (int32_t)std::max<int64_t>(std::max<int64_t>(nblk, ext.ptr ? 0 : blk_cap), 1);
  const size_t n_blk = tau > 0.0f ? (size_t)n_seqs * H * a->blk_stride * 8 : 0;
  // sparse-V gather: the candidate blocks' scores (16 per block row and
  // head) after the maxima, then one arrival counter per (sequence, q head);
  // without room for them in a caller's scratch, the gated pass
  bool gather = tau > 0.0f && g_sparse_gather && nblk <= fmkv::kGatherMaxRows;
  const size_t score_off = blk_off + n_blk;  // a multiple of 4 floats
  const size_t cnt_off = score_off + 16 * n_blk;
  const size_t need_gather = (cnt_off + (size_t)n_seqs * n_q_heads) * sizeof(float);
  if (gather && ext.ptr && need_gather > ext.bytes) gather = false;
  const size_t need =
      gather ? need_gather : (n_blk ? blk_off + n_blk : stat_off + n_stat_ml) * sizeof(float);
  float* ws = ext.ptr;
  if (ws) {
    if (need > ext.bytes)
      return fail(FMKV_ERR_CAPACITY, "this call needs " + std::to_string(need) +
                                         " bytes of split partials; the no-allocation scratch "
                                         "holds " + std::to_string(ext.bytes));
  } else {
    // One cache: the workspace is sized once for the largest plan the
    // cache's capacity allows (split count at most the planned work-groups
    // per KV head + 1, a new-token column, sparse-V statistics and block
    // maxima), so that it does not grow as the context does and a decode
    // step captured into a HIP graph stays valid. A paged batch's need
    // depends on each call's batch and grows on demand.
    size_t alloc = need;
    if (n_seqs == 1 && !st.block_table) {
      const int64_t per_head = ((int64_t)wg_per_cu * o->cus + H - 1) / H + 1;
      const int64_t max_splits =
          std::max<int64_t>(g_bps_override > 0 ? blk_cap : std::min<int64_t>(blk_cap, per_head),
                            a->max_splits);
      const size_t rows = (size_t)(max_splits + 1) * n_q_heads;
      const size_t off = (rows * (D + 2) + 3 * (size_t)n_q_heads + 2 * rows + 3) & ~(size_t)3;
      const size_t blks = (size_t)H * std::max<int64_t>(std::max<int64_t>(blk_cap, nblk), 1) * 8;
      alloc = std::max(need, (off + blks * (gather ? 17 : 1) + (gather ? n_q_heads : 0)) * sizeof(float));
    }
    rc = o->ws.ensure(alloc);
    if (rc) return rc;
    ws = o->ws.ptr;
  }
  a->part_o = n_rows ? ws : nullptr;
  a->part_ml = n_rows ? ws + n_rows * D : nullptr;
  a->tau_stats = n_stats ? ws + n_rows * (D + 2) : nullptr;
  a->stat_ml = n_stat_ml ? ws + stat_off : nullptr;
  a->blk_max = n_blk ? ws + blk_off : nullptr;
  a->blk_scores = gather ? ws + score_off : nullptr;
  a->sv_count = gather ? reinterpret_cast<int32_t*>(ws + cnt_off) : nullptr;
  if (gather) {
    // parts per (sequence, q head): the kept tokens, and so the candidate
    // blocks, are at most min(visible tokens, 1 / tau); one part per 128 of
    // them, at most 64 (the gather uses one per 16 candidate blocks)
    const double inv_tau = std::ceil(1.0 / (double)tau);
    const int64_t bound = std::min<int64_t>(nblk * fmkv::kBlockTokens,
                                            inv_tau < 1e15 ? (int64_t)inv_tau : INT64_MAX);
    a->gather_parts = (int32_t)std::clamp<int64_t>((bound + 127) / 128, 1,
                                                   std::min<int64_t>(a->part_stride, 16));
    a->gather_rows = (int32_t)std::max<int64_t>(nblk, 1);
  }
  return FMKV_OK;
}

// Decode attention over the first T positions of a cache.
int prepare_attention(fmkv_cache* c, int64_t T, const void* q, int32_t n_q_heads, float scale,
                      float tau, void* out, int32_t out_dtype, int new_col, fmkv::AttnArgs* a,
                      ExtWorkspace ext = {}) {
  // a ring's slots; its visible positions are the last `window` of the T,
  // which the kernels test per slot whenever that hides stored slots
  const int64_t W = ring_slots(c->desc);
  a->seq_lens = nullptr;
  a->seq_len = T;
  a->window = W;
  a->vis_begin = W > 0 ? std::max<int64_t>(c->vis_begin, T - c->desc.window) : c->vis_begin;
  const int64_t filled = W > 0 ? std::min<int64_t>(T, W) : T;
  const int64_t vb = W > 0 ? 0 : c->vis_begin;
  const int64_t nblk =
      (filled + fmkv::kBlockTokens - 1) / fmkv::kBlockTokens - vb / fmkv::kBlockTokens;
  const int wg_per_cu = attn_wg_per_cu(c->desc);
  const int64_t blk_cap = n_slots_of(c->desc) / fmkv::kBlockTokens;
  return prepare_attention_common(c, cache_store(c), 1, nblk, blk_cap, q, n_q_heads, scale, tau,
                                  out, out_dtype, wg_per_cu, 1, 1, new_col, a, ext);
}

// The most blocks that hold a window of `win` positions and `sinks` first ones.
int64_t window_blocks(int64_t win, int64_t sinks) {
  constexpr int64_t B = fmkv::kBlockTokens;
  return (win + B - 2) / B + 1 + (sinks + B - 1) / B;
}

// A window's arguments; the GPU of a call.
int check_window(int32_t window, int32_t sinks) {
  if (window < 1 || window > (1 << 30))
    return fail(FMKV_ERR_INVALID_ARG, "window must be in [1, 2^30]");
  if (sinks < 0 || sinks > (1 << 30)) return fail(FMKV_ERR_INVALID_ARG, "sinks must be in [0, 2^30]");
  return FMKV_OK;
}
int check_device(const fmkv_pool* p) {
  int dev = -1;
  const hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
  if (dev != p->device)
    return fail(FMKV_ERR_INVALID_ARG, "the pool is on GPU " + std::to_string(p->device) +
                                          ", the current GPU is " + std::to_string(dev));
  return FMKV_OK;
}

int prepare_paged_append(const fmkv_pool* p, const void* k, const void* v,
                         const int32_t* block_tables, int32_t max_blocks, const int32_t* start_pos,
                         int32_t n_seqs, int32_t n_new, fmkv::AppendArgs* a, int* tasks) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  if (n_seqs < 0 || n_new < 0 || max_blocks < 1)
    return fail(FMKV_ERR_INVALID_ARG, "n_seqs/n_new must be >= 0 and max_blocks >= 1");
  if (n_seqs == 0 || n_new == 0) return FMKV_OK;
  if (!k || !v || !block_tables || !start_pos)
    return fail(FMKV_ERR_INVALID_ARG, "k/v/block_tables/start_pos must be device pointers");
  if (n_seqs > 65535) return fail(FMKV_ERR_INVALID_ARG, "at most 65535 sequences per call");
  a->st = pool_store(p, block_tables, max_blocks);
  a->k = static_cast<const uint16_t*>(k);
  a->v = static_cast<const uint16_t*>(v);
  a->start_pos = start_pos;
  a->start_scalar = 0;
  a->n_new = n_new;
  a->window = 0;
  std::memcpy(a->sign_bits, p->sign_bits, sizeof(a->sign_bits));
  a->c = p->c;
  a->sqrt_d = p->sqrt_d;
  a->cb_bits = p->desc.bits;
  *tasks =(n_new + fmkv::kBlockTokens - 1) / fmkv::kBlockTokens + 1;
  return FMKV_OK;
}

// Blocks per split of a window's call: nblk visible blocks at most for each of
// `rows` (sequence, KV head) pairs. A split costs its blocks and a fixed part (q
// table, merge of its streams: about 12 blocks' time, 3 of the plain kernel's),
// each round of work-groups that the chip takes at once costs the longest split
// in it, every split a tenth of a block in the combine, and the combine's launch
// as much as the fixed part (one split a sequence has none). So the splits of
// each number of rounds are as many as fit it, or as the combine allows, and
// equal; the cheapest wins. (us per call, by blocks per split: one sequence,
// 66 blocks of 4 bits, 256 dims, 8 heads: 1: 20.1, 2: 15.4, 3: 10.9, 8: 11.0, 16:
// 13.0; seven of 254 blocks each, 8 bits, 512 dims, 2 heads: 14, which leaves 10
// work-groups to a second round: 28.7, 15, what this comes to: 23.6, 16: 23.0, 32:
// 27.1; seven ragged ones within that bound, whose short ones leave room in the
// first round: 14: 21.2, 15: 21.9, 16: 21.4; 32 ragged ones of up
// to 258 blocks, 4 bits: 64 (4 splits and one of 2 blocks): 60.2, 86: 51.4, 129:
// 53.9; the same all at 258: 66.5, 65.7, 63.9; one of 254 blocks, 2 heads of 512
// dims: 2: 17.0, 4: 15.5, 8: 16.8, 16: 19.6.)
int64_t window_bps(const fmkv_cache_desc& d, int cus, int64_t nblk, int64_t rows, int new_col) {
  if (nblk < 1) return 1;
  const bool plain = d.mode == FMKV_MODE_PLAIN;
  const double fixed = plain ? 3.0 : 12.0;
  const int64_t few = std::max<int64_t>((int64_t)std::sqrt(10.0 * (double)nblk), 1);
  auto best = [&](int64_t per_cu, int64_t min_bps) {
    int64_t slots = per_cu * cus;
    if (new_col && rows <= slots / 2) slots -= rows;  // the new-token column's work-groups
    int64_t bps = 0;
    double cost = 0.0;
    const int64_t r0 = (rows + slots - 1) / slots;
    for (int64_t r = r0; r < r0 + 4; r++) {
      const int64_t s = std::clamp<int64_t>(r * slots / rows, 1, std::min(few, nblk));
      const int64_t b = std::max((nblk + s - 1) / s, min_bps), n = (nblk + b - 1) / b;
      const double c = (double)((n * rows + slots - 1) / slots) * ((double)b + fixed) + 0.1 * (double)n +
                       (n > 1 || new_col ? fixed : 0.0);
      if (bps == 0 || c < cost) bps = b, cost = c;
    }
    return bps;
  };
  // (the plain kernel's registers: five work-groups a CU, at 512 dims three, of
  // which two are counted: 32 sequences of 66 blocks, 8 heads of 256 dims: five
  // splits 57.2 us, two 64.8; 64 sequences, 2 heads of 512 dims: four splits 66.0,
  // six 70.4)
  if (plain) return best(d.head_dim == 512 ? 2 : 5, 1);
  if (paged_solo_slots(d) == 1) return best(1, 1);
  // wave pairs, one work-group per CU, while a round of them is enough; else
  // single-wave streams, three per CU
  const int64_t pairs = best(1, 1);
  return pairs < 8 && (nblk + pairs - 1) / pairs * rows <= cus ? pairs : best(3, 8);
}

// win > 0: over the last `win` positions and the first `sinks` ones.
int prepare_paged_attention(fmkv_pool* p, const void* q, const int32_t* block_tables,
                            int32_t max_blocks, const int32_t* seq_lens, int32_t n_seqs,
                            int32_t max_seq_len, int32_t n_q_heads, float scale, float tau,
                            void* out, int32_t out_dtype, int new_col, hipStream_t s,
                            fmkv::AttnArgs* a, int32_t win = 0, int32_t sinks = 0) {
  if (n_seqs < 0 || max_seq_len < 0 || max_blocks < 1)
    return fail(FMKV_ERR_INVALID_ARG, "bad n_seqs / max_seq_len / max_blocks");
  if (n_seqs > 0 && (!block_tables || !seq_lens))
    return fail(FMKV_ERR_INVALID_ARG, "block_tables/seq_lens are null");
  if ((int64_t)max_seq_len > (int64_t)max_blocks * fmkv::kBlockTokens)
    return fail(FMKV_ERR_INVALID_ARG, "max_seq_len exceeds max_blocks * 16");
  if (n_seqs > 65535) return fail(FMKV_ERR_INVALID_ARG, "at most 65535 sequences per call");
  RelaxedCapture relaxed;  // (the workspace may grow)
  p->ws.captured = is_captured(s);
  a->seq_lens = seq_lens;
  a->seq_len = 0;
  a->window = 0;
  a->vis_begin = 0;
  if (win > 0) {
    if (n_seqs == 0) return FMKV_OK;
    int rc = check_attn_args(p->desc, q, n_q_heads, tau, out, out_dtype);
    if (rc) return rc;
    // (a copy to LDS in pieces of 16 bytes, whose last address bits do not count)
    if ((uintptr_t)q % 16 != 0) return fail(FMKV_ERR_UNSUPPORTED, "q must be 16-byte aligned");
    if ((rc = check_device(p))) return rc;
  }
  a->win = win;
  a->sinks = sinks;
  int64_t nblk = ((int64_t)max_seq_len + fmkv::kBlockTokens - 1) / fmkv::kBlockTokens;
  if (win > 0) nblk = std::min(nblk, window_blocks(win, sinks));
  // Ragged lengths: the bound counts every sequence at max_seq_len, so the
  // plan aims at several work-groups per CU (the dispatcher balances their
  // uneven sizes), but at least 64 blocks each (a work-group's prologue and
  // epilogue cost about as much as a dozen blocks) -- unless that would
  // leave CUs idle: the floor never exceeds one CU's share of all blocks,
  // so a small batch at long context still spreads over every CU. When the
  // grid holds at least four work-groups per CU, each sequence's first split
  // is four times larger: the big work-groups start first and the small
  // ones fill the tail (32 sequences of 512..16384 tokens: bps 171, 197 us;
  // equal splits at four per CU: 207 us). A grid of fewer work-groups has
  // no tail to fill, and a larger first split would only end last.
  //
  // Affine head-blocks of at most 1024 code bits per token (head_dim 128,
  // head_dim 256 at 4 bits) run as work-groups of four single-wave streams,
  // three to a CU (slots = 3): the plan counts slots instead of CUs, six
  // work-groups per slot, and the floor is at most one slot's share (one
  // sequence of 65536 tokens, Hkv 8, head_dim 256, 4 bits: bps 43, one
  // work-group per slot, 40.7 us; bps 22 or 128: 47.6 / 52.5 us; the 32
  // ragged sequences above at bps 57..96: 173-178 us, against 202 us with
  // twelve-wave work-groups, one per CU).
  const int n_s = n_seqs > 0 ? n_seqs : 1;
  const int64_t total = nblk * p->desc.n_kv_heads * n_s;
  const int slots = paged_solo_slots(p->desc);
  const int64_t n_slots = (int64_t)slots * p->cus;
  const int64_t share = (total + n_slots - 1) / n_slots;
  const int min_bps = (int)std::min<int64_t>(64, std::max<int64_t>(share, 1));
  const int wg_per_cu = 6 * slots * fmkv::kAttnWgPerCu;
  if (win > 0) {
    const int64_t b = window_bps(p->desc, p->cus, nblk, (int64_t)p->desc.n_kv_heads * n_s, new_col);
    return prepare_attention_common(p, pool_store(p, block_tables, max_blocks), n_s, nblk,
                                    max_blocks, q, n_q_heads, scale, tau, out, out_dtype,
                                    1 << 20 /* b is the blocks per split */, (int)b, 1, new_col, a);
  }
  const int64_t bps = choose_bps(total, p->cus, wg_per_cu, 0, min_bps);
  const int first_mult = total >= 4 * n_slots * bps ? 4 : 1;
  return prepare_attention_common(p, pool_store(p, block_tables, max_blocks), n_s, nblk,
                                  max_blocks, q, n_q_heads, scale, tau, out, out_dtype, wg_per_cu,
                                  min_bps, first_mult, new_col, a);
}

int decode_step_impl(fmkv_cache* c, const void* k, const void* v, int64_t n, const void* q,
                     int32_t n_q_heads, float scale, float tau, void* out, int32_t out_dtype,
                     void* stream, ExtWorkspace ext, const fmkv_kv_prologue* pro = nullptr);

// The prologue on the decode step's new-token column (a fused step).
void set_prologue(const fmkv_kv_prologue* pro, fmkv::AttnArgs* a) {
  a->k_norm_w = static_cast<const uint16_t*>(pro->k_norm_weight);
  a->eps = pro->eps;
  a->rope_dims = pro->rope_dims;
  a->rope_theta = pro->rope_theta;
}

// The decode attention kernel of the cache's mode (and the split combine).
hipError_t launch_attention(const fmkv::AttnArgs& a, int n_seqs, int n_kv_heads, hipStream_t s,
                            hipEvent_t e0, hipEvent_t e1) {
  if (a.st.layout.mode == fmkv::kCodebook)
    return fmkv::launch_cb_decode_attention(a, n_seqs, n_kv_heads, s, e0, e1);
  if (a.st.layout.mode == fmkv::kPlain)
    return fmkv::launch_plain_decode_attention(a, n_seqs, n_kv_heads, s, e0, e1);
  return fmkv::launch_decode_attention(a, n_seqs, n_kv_heads, s, e0, e1);
}

}  // namespace

// Device memory of fmkv_decode_step_noalloc: the split partials (and
// sparse-V statistics) of one decode step, as the handle's workspace holds
// them for fmkv_decode_step. Every GPU holds its own copy for the life of the
// process; in host code the name only stands in for it, so the library takes
// each device's address once (noalloc_scratch) and passes that address on.
// The lookup runs at set-up, when a cache handle is created on the device:
// the runtime materialises the symbol's storage on the first lookup (about
// 10 MiB of device memory on one MI355X), which the allocation-free entry
// point must not do. Calls on one GPU share it: every call writes what it
// reads before reading it, and calls that overlap in time on one GPU race.
static __device__ __align__(256) uint8_t scratch[FMKV_NOALLOC_SCRATCH_BYTES];

namespace {

std::mutex g_scratch_mu;
void* g_scratch_dev[kMaxDevices] = {};

// This device's address of `scratch`, looked up once per device with the
// device current (hipGetSymbolAddress allocates nothing).
int noalloc_scratch(ExtWorkspace* out) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(FMKV_ERR_UNSUPPORTED, "device index beyond 63");
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_dev[dev]) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !p) return hip_fail(e, "hipGetSymbolAddress(scratch)");
    g_scratch_dev[dev] = p;
  }
  out->ptr = static_cast<float*>(g_scratch_dev[dev]);
  out->bytes = FMKV_NOALLOC_SCRATCH_BYTES;
  return FMKV_OK;
}

}  // namespace

extern "C" {

const char* fmkv_last_error(void) { return g_err.c_str(); }

int fmkv_validate_desc(const fmkv_cache_desc* desc) { return check_desc(desc); }

int fmkv_layout_bytes(const fmkv_cache_desc* desc, int64_t* block_bytes, int64_t* arena_bytes) {
  int rc = check_desc(desc);
  if (rc) return rc;
  const BlockLayout L = fmkv::make_layout(desc->head_dim, desc->bits, desc->mode);
  if (block_bytes) *block_bytes = L.block_bytes;
  if (arena_bytes)
    *arena_bytes = L.block_bytes * desc->n_kv_heads * (n_slots_of(*desc) / fmkv::kBlockTokens);
  return FMKV_OK;
}

int fmkv_cache_create(const fmkv_cache_desc* desc, fmkv_cache** out) {
  int rc = check_desc(desc);
  if (rc) return rc;
  if (!out) return fail(FMKV_ERR_INVALID_ARG, "out is null");
  *out = nullptr;
  fmkv_cache* c = new fmkv_cache();
  c->desc = *desc;
  c->layout = fmkv::make_layout(desc->head_dim, desc->bits, desc->mode);
  c->n_blocks = n_slots_of(*desc) / fmkv::kBlockTokens;
  c->c = 1.0f / std::sqrt((float)desc->head_dim);
  c->sqrt_d = std::sqrt((float)desc->head_dim);
  c->offset = 0;
  c->vis_begin = 0;
  c->arena = nullptr;
  c->d_signs = nullptr;
  const int64_t bytes = c->layout.block_bytes * c->n_blocks * desc->n_kv_heads;
  hipError_t e = hipMalloc(&c->arena, bytes);
  if (e != hipSuccess) {
    delete c;
    return fail(FMKV_ERR_OOM, "cache arena allocation failed (" + std::to_string(bytes) + " bytes)");
  }
  e = hipMemset(c->arena, 0, bytes);
  if (e != hipSuccess) {
    (void)hipFree(c->arena);
    delete c;
    return hip_fail(e, "hipMemset(arena)");
  }
  rc = make_signs(*desc, &c->d_signs);
  if (rc) {
    (void)hipFree(c->arena);
    delete c;
    return rc;
  }
  sign_bits_of(*desc, c->sign_bits);
  c->cus = device_cus();
  c->split = prefill_scratch_join();
  // set-up of the no-allocation decode step's scratch on this device (once
  // per device; later creations find the address recorded)
  ExtWorkspace ext;
  rc = noalloc_scratch(&ext);
  if (rc) {
    (void)fmkv_cache_destroy(c);
    return rc;
  }
  *out = c;
  return FMKV_OK;
}

int fmkv_cache_destroy(fmkv_cache* c) {
  if (!c) return FMKV_OK;
  if (c->arena) (void)hipFree(c->arena);
  if (c->d_signs) (void)hipFree(c->d_signs);
  c->ws.release();
  c->stage.release();
  prefill_scratch_leave(c->split);
  delete c;
  return FMKV_OK;
}

int fmkv_cache_offset(const fmkv_cache* c, int64_t* out) {
  if (!c || !out) return fail(FMKV_ERR_INVALID_ARG, "null argument");
  *out = c->offset;
  return FMKV_OK;
}

int fmkv_cache_stored_len(const fmkv_cache* c, int64_t* out) {
  if (!c || !out) return fail(FMKV_ERR_INVALID_ARG, "null argument");
  *out = c->offset - visible_begin(c);
  return FMKV_OK;
}

int fmkv_cache_append(fmkv_cache* c, const void* k, const void* v, int64_t n, void* stream) {
  fmkv::AppendArgs a;
  int64_t tasks = 0;
  int rc = prepare_append(c, k, v, n, &a, &tasks);
  if (rc || n == 0) return rc;
  hipError_t e = fmkv::launch_append(a, 1, (int)tasks, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "append launch");
  c->offset += n;
  return FMKV_OK;
}

int fmkv_cache_append_projected(fmkv_cache* c, const void* k, const void* v, int64_t n,
                                const fmkv_kv_prologue* pro, void* stream) {
  if (!c) return fail(FMKV_ERR_INVALID_ARG, "cache is null");
  int rc = check_prologue(c->desc, pro);
  if (rc) return rc;
  fmkv::AppendArgs a;
  int64_t tasks = 0;
  rc = prepare_append(c, k, pro->v_from_k ? k : v, n, &a, &tasks);
  if (rc || n == 0) return rc;
  set_prologue(pro, &a);
  hipError_t e = fmkv::launch_append(a, 1, (int)tasks, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "append launch");
  c->offset += n;
  return FMKV_OK;
}

int fmkv_prefill_step(fmkv_cache* c, const void* k, const void* v, int64_t n, const void* q,
                      int32_t n_q_heads, float scale, void* out, int32_t out_dtype, void* stream) {
  if (!c) return fail(FMKV_ERR_INVALID_ARG, "cache is null");
  if (n < 1) return fail(FMKV_ERR_INVALID_ARG, "a prefill step appends at least one token");
  int rc = check_attn_args(c->desc, q, n_q_heads, 0.0f, out, out_dtype);
  if (rc) return rc;
  if (!std::isfinite(scale)) return fail(FMKV_ERR_INVALID_ARG, "scale must be finite");
  const int32_t group = n_q_heads / c->desc.n_kv_heads;
  if (n > (int64_t)65535 * (64 / group))
    return fail(FMKV_ERR_INVALID_ARG, "n_tokens too large for one prefill step");
  fmkv::AppendArgs ap;
  int64_t tasks = 0;
  rc = prepare_append(c, k, v, n, &ap, &tasks);
  if (rc) return rc;
  const int64_t p0 = c->offset, W = c->desc.window;  // the sliding window (0: causal only)
  const int H = c->desc.n_kv_heads;
  const int64_t bb = c->layout.block_bytes;
  fmkv::PrefillArgs pa;
  pa.old_st = cache_store(c);
  pa.new_st = pa.old_st;
  pa.p0 = p0;
  pa.start_pos = nullptr;
  pa.n_seqs = 1;
  pa.n_q = (int32_t)n;
  pa.window = W;
  pa.ring_slots = ring_slots(c->desc);
  pa.vis_begin = c->vis_begin;
  pa.p_split = 0;
  pa.new_blk0 = 0;
  pa.group = group;
  pa.n_q_heads = n_q_heads;
  pa.q = static_cast<const uint16_t*>(q);
  pa.qscale = scale * 1.4426950408889634f;
  std::memcpy(pa.sign_bits, c->sign_bits, sizeof(pa.sign_bits));
  pa.c = c->c;
  pa.out = out;
  pa.out_f32 = out_dtype == FMKV_DTYPE_F32 ? 1 : 0;
  fmkv::AppendArgs as = ap;
  int64_t nsb = 0;
  if (W > 0) {
    // the chunk's rows go to a staging store first (block 0 = absolute
    // block p0 / 16), so the ring keeps every position the queries need
    nsb = (p0 % fmkv::kBlockTokens + n + fmkv::kBlockTokens - 1) / fmkv::kBlockTokens;
    rc = c->stage.ensure((size_t)(nsb * H * bb), true);
    if (rc) return rc;
    fmkv::Store st;
    st.base = reinterpret_cast<uint8_t*>(c->stage.ptr);
    st.block_stride = bb;
    st.head_stride = nsb * bb;
    st.block_table = nullptr;
    st.table_stride = 0;
    st.n_blocks = nsb;
    st.n_kv_heads = H;
    st.layout = c->layout;
    as.st = st;
    as.start_scalar = p0 % fmkv::kBlockTokens;
    as.window = 0;
    pa.new_st = st;
    pa.p_split = p0;
    pa.new_blk0 = p0 / fmkv::kBlockTokens;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e;
  int64_t keys = p0 + n - c->vis_begin;
  if (W > 0 && keys > W + 64) keys = W + 64;
  const int64_t max_steps = keys / 32 + 2;
  if (W > 0) {
    e = fmkv::launch_append(as, 1, (int)nsb, s);
    if (e != hipSuccess) return hip_fail(e, "staging append launch");
    e = run_prefill(pa, c->split, c->cus, max_steps, s);
    if (e != hipSuccess) return hip_fail(e, "prefill attention launch");
    e = fmkv::launch_append(ap, 1, (int)tasks, s);
    if (e != hipSuccess) return hip_fail(e, "append launch");
  } else {
    e = fmkv::launch_append(ap, 1, (int)tasks, s);
    if (e != hipSuccess) return hip_fail(e, "append launch");
    e = run_prefill(pa, c->split, c->cus, max_steps, s);
    if (e != hipSuccess) return hip_fail(e, "prefill attention launch");
  }
  c->offset += n;
  return FMKV_OK;
}

int fmkv_decode_step(fmkv_cache* c, const void* k, const void* v, int64_t n, const void* q,
                     int32_t n_q_heads, float scale, float tau, void* out, int32_t out_dtype,
                     void* stream) {
  return decode_step_impl(c, k, v, n, q, n_q_heads, scale, tau, out, out_dtype, stream, {});
}

int fmkv_decode_step_projected(fmkv_cache* c, const void* k_proj, const void* v_proj, int64_t n,
                               const fmkv_kv_prologue* pro, const void* q, int32_t n_q_heads,
                               float scale, float tau, void* out, int32_t out_dtype, void* stream) {
  if (!pro) return fail(FMKV_ERR_INVALID_ARG, "prologue is null");
  return decode_step_impl(c, k_proj, v_proj, n, q, n_q_heads, scale, tau, out, out_dtype, stream,
                          {}, pro);
}

int fmkv_decode_step_noalloc(fmkv_cache* c, const void* k, const void* v, int64_t n,
                             const void* q, int32_t n_q_heads, float scale, float tau, void* out,
                             int32_t out_dtype, void* stream) {
  if (!c) return fail(FMKV_ERR_INVALID_ARG, "cache is null");
  ExtWorkspace ext;
  int rc = noalloc_scratch(&ext);
  if (rc) return rc;
  return decode_step_impl(c, k, v, n, q, n_q_heads, scale, tau, out, out_dtype, stream, ext);
}

}  // extern "C"

namespace {

int decode_step_impl(fmkv_cache* c, const void* k, const void* v, int64_t n, const void* q,
                     int32_t n_q_heads, float scale, float tau, void* out, int32_t out_dtype,
                     void* stream, ExtWorkspace ext, const fmkv_kv_prologue* pro) {
  if (!c) return fail(FMKV_ERR_INVALID_ARG, "cache is null");
  if (n < 1) return fail(FMKV_ERR_INVALID_ARG, "a decode step appends at least one token");
  int rc;
  if (pro && (rc = check_prologue(c->desc, pro))) return rc;
  fmkv::AppendArgs ap;
  int64_t tasks = 0;
  rc = prepare_append(c, k, pro && pro->v_from_k ? k : v, n, &ap, &tasks);
  if (rc) return rc;
  if (pro) set_prologue(pro, &ap);
  // one new token: the attention launch appends it itself (new-token
  // column; with sparse-V the statistics pass does); chunks append first
  const int fused = n == 1 ? 1 : 0;
  fmkv::AttnArgs at;
  rc = prepare_attention(c, c->offset + n, q, n_q_heads, scale, tau, out, out_dtype, fused, &at, ext);
  if (rc) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e;
  if (fused) {
    at.k_new = ap.k;
    at.v_new = ap.v;
    if (pro) set_prologue(pro, &at);
  } else {
    e = fmkv::launch_append(ap, 1, (int)tasks, s);
    if (e != hipSuccess) return hip_fail(e, "append launch");
    c->offset += n;
  }
  hipEvent_t e0, e1;
  next_events(&e0, &e1);
  e = launch_attention(at, 1, c->desc.n_kv_heads, s, e0, e1);
  if (e != hipSuccess) return hip_fail(e, "decode attention launch");
  if (fused) c->offset += n;
  return FMKV_OK;
}

// Elapsed milliseconds of recorded pair i (waits for it).
int profile_pair_ms(int32_t i, float* ms) {
  hipError_t e = hipEventSynchronize(g_prof.ev[2 * (size_t)i + 1]);
  if (e != hipSuccess) return hip_fail(e, "hipEventSynchronize");
  *ms = 0.0f;
  e = hipEventElapsedTime(ms, g_prof.ev[2 * (size_t)i], g_prof.ev[2 * (size_t)i + 1]);
  if (e != hipSuccess) return hip_fail(e, "hipEventElapsedTime");
  return FMKV_OK;
}

}  // namespace

extern "C" {

int fmkv_cache_trim(fmkv_cache* c, int64_t keep_last) {
  if (!c) return fail(FMKV_ERR_INVALID_ARG, "cache is null");
  if (keep_last < 0) return fail(FMKV_ERR_INVALID_ARG, "keep_last must be >= 0");
  const int64_t b = c->offset - keep_last;
  if (b > c->vis_begin) c->vis_begin = b;
  return FMKV_OK;
}

int fmkv_decode_attention(fmkv_cache* c, const void* q, int32_t n_q_heads, float scale, float tau,
                          void* out, int32_t out_dtype, void* stream) {
  if (!c) return fail(FMKV_ERR_INVALID_ARG, "cache is null");
  fmkv::AttnArgs a;
  int rc = prepare_attention(c, c->offset, q, n_q_heads, scale, tau, out, out_dtype, 0, &a);
  if (rc) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipEvent_t e0, e1;
  next_events(&e0, &e1);
  hipError_t e = launch_attention(a, 1, c->desc.n_kv_heads, s, e0, e1);
  if (e != hipSuccess) return hip_fail(e, "decode attention launch");
  return FMKV_OK;
}

int fmkv_cache_decode_splits(const fmkv_cache* c, int32_t* n_splits) {
  if (!c || !n_splits) return fail(FMKV_ERR_INVALID_ARG, "null argument");
  int64_t filled = c->desc.window > 0 ? std::min<int64_t>(c->offset, ring_slots(c->desc)) : c->offset;
  int64_t vb = c->desc.window > 0 ? 0 : c->vis_begin;
  int64_t nblk = (filled + fmkv::kBlockTokens - 1) / fmkv::kBlockTokens - vb / fmkv::kBlockTokens;
  if (nblk < 1) nblk = 1;
  fmkv::AttnArgs a;
  plan_splits(c->cus, c->desc.n_kv_heads, 1, nblk, attn_wg_per_cu(c->desc), 1, 1, 0, false, &a);
  *n_splits = a.max_splits;
  return FMKV_OK;
}

int fmkv_cache_fetch(const fmkv_cache* c, void* k_out, void* v_out, int32_t out_dtype, void* stream) {
  if (!c) return fail(FMKV_ERR_INVALID_ARG, "cache is null");
  if (!k_out || !v_out) return fail(FMKV_ERR_INVALID_ARG, "k_out/v_out must be device pointers");
  if (out_dtype != FMKV_DTYPE_BF16 && out_dtype != FMKV_DTYPE_F32)
    return fail(FMKV_ERR_INVALID_ARG, "bad out_dtype");
  fmkv::FetchArgs a;
  a.st = cache_store(c);
  a.offset = c->offset;
  a.window = ring_slots(c->desc);  // slot of position p: p mod the ring's slots
  a.first_pos = visible_begin(c);
  a.n_pos = c->offset - a.first_pos;
  a.signs = c->d_signs;
  a.c = c->c;
  a.k_out = k_out;
  a.v_out = v_out;
  a.out_f32 = out_dtype == FMKV_DTYPE_F32;
  hipError_t e = fmkv::launch_fetch(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "fetch launch");
  return FMKV_OK;
}

int fmkv_cache_read_codes(const fmkv_cache* c, void* codes, void* meta, void* stream) {
  if (!c) return fail(FMKV_ERR_INVALID_ARG, "cache is null");
  if (!codes || (!meta && c->desc.mode != FMKV_MODE_PLAIN))
    return fail(FMKV_ERR_INVALID_ARG, "codes/meta must be device pointers");
  fmkv::ReadArgs a;
  a.st = cache_store(c);
  a.n_slots = c->desc.window > 0 ? ring_slots(c->desc) : c->desc.capacity;
  a.codes = static_cast<uint32_t*>(codes);
  a.meta = static_cast<uint16_t*>(meta);
  hipError_t e = fmkv::launch_read_codes(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "read_codes launch");
  return FMKV_OK;
}

int fmkv_pool_create(const fmkv_cache_desc* desc, int64_t n_blocks, fmkv_pool** out) {
  if (!desc) return fail(FMKV_ERR_INVALID_ARG, "descriptor is null");
  fmkv_cache_desc d = *desc;
  d.window = 0;
  d.capacity = 1;
  int rc = check_desc(&d);
  if (rc) return rc;
  if (desc->window != 0) return fail(FMKV_ERR_UNSUPPORTED, "paged pools hold global (linear) sequences");
  if (!out) return fail(FMKV_ERR_INVALID_ARG, "out is null");
  if (n_blocks < 1 || n_blocks > ((int64_t)1 << 31) - 1)
    return fail(FMKV_ERR_INVALID_ARG, "n_blocks must be in [1, 2^31)");
  *out = nullptr;
  fmkv_pool* p = new fmkv_pool();
  p->desc = *desc;
  p->layout = fmkv::make_layout(desc->head_dim, desc->bits, desc->mode);
  p->n_blocks = n_blocks;
  p->c = 1.0f / std::sqrt((float)desc->head_dim);
  p->sqrt_d = std::sqrt((float)desc->head_dim);
  p->arena = nullptr;
  p->d_signs = nullptr;
  const int64_t bytes = p->layout.block_bytes * desc->n_kv_heads * n_blocks;
  hipError_t e = hipMalloc(&p->arena, bytes);
  if (e != hipSuccess) {
    delete p;
    return fail(FMKV_ERR_OOM, "pool allocation failed (" + std::to_string(bytes) + " bytes)");
  }
  e = hipMemset(p->arena, 0, bytes);
  if (e != hipSuccess) {
    (void)hipFree(p->arena);
    delete p;
    return hip_fail(e, "hipMemset(pool)");
  }
  rc = make_signs(*desc, &p->d_signs);
  if (rc) {
    (void)hipFree(p->arena);
    delete p;
    return rc;
  }
  sign_bits_of(*desc, p->sign_bits);
  p->cus = device_cus();
  p->split = prefill_scratch_join();
  p->device = 0;
  (void)hipGetDevice(&p->device);
  *out = p;
  return FMKV_OK;
}

int fmkv_pool_destroy(fmkv_pool* p) {
  if (!p) return FMKV_OK;
  if (p->arena) (void)hipFree(p->arena);
  if (p->d_signs) (void)hipFree(p->d_signs);
  p->ws.release();
  prefill_scratch_leave(p->split);
  delete p;
  return FMKV_OK;
}

int fmkv_paged_prefill_step(fmkv_pool* p, const void* k, const void* v,
                            const int32_t* block_tables, int32_t max_blocks,
                            const int32_t* start_pos, int32_t n_seqs, int32_t n_new,
                            const void* q, int32_t n_q_heads, float scale, void* out,
                            int32_t out_dtype, void* stream) {
  return fmkv_paged_prefill_step_bounded(p, k, v, block_tables, max_blocks, start_pos, n_seqs,
                                         n_new, 0, q, n_q_heads, scale, out, out_dtype, stream);
}

}  // extern "C"

namespace {

// Batched prefill: the append of k and v (both null with `stored`: the rows are
// in the pool), then the attention, over a window with sinks where window > 0.
int paged_prefill_impl(fmkv_pool* p, bool stored, const void* k, const void* v,
                       const int32_t* block_tables, int32_t max_blocks, const int32_t* start_pos,
                       int32_t n_seqs, int32_t n_new, int32_t max_seq_len, const void* q,
                       int32_t n_q_heads, float scale, int32_t window, int32_t sinks, void* out,
                       int32_t out_dtype, void* stream) {
  if (max_seq_len < 0) return fail(FMKV_ERR_INVALID_ARG, "max_seq_len must be >= 0 (0: unknown)");
  if (n_seqs < 1 || n_new < 1)
    return fail(FMKV_ERR_INVALID_ARG, "a prefill step needs n_seqs >= 1 and n_new >= 1");
  int rc = check_attn_args(p->desc, q, n_q_heads, 0.0f, out, out_dtype);
  if (rc) return rc;
  if (!std::isfinite(scale)) return fail(FMKV_ERR_INVALID_ARG, "scale must be finite");
  const int32_t group = n_q_heads / p->desc.n_kv_heads;
  if ((int64_t)n_new > (int64_t)65535 * (64 / group))
    return fail(FMKV_ERR_INVALID_ARG, "n_new too large for one prefill step");
  fmkv::AppendArgs ap;
  int tasks = 0;
  // (stored: q stands in for the rows, which are not read)
  rc = prepare_paged_append(p, stored ? q : k, stored ? q : v, block_tables, max_blocks, start_pos,
                            n_seqs, n_new, &ap, &tasks);
  if (rc) return rc;
  if (window > 0 && (rc = check_device(p))) return rc;
  fmkv::PrefillArgs pa;
  pa.old_st = ap.st;
  pa.new_st = ap.st;
  pa.sinks = sinks;
  pa.p0 = 0;
  pa.start_pos = start_pos;
  pa.n_seqs = n_seqs;
  pa.n_q = n_new;
  pa.window = window;
  pa.ring_slots = 0;
  pa.vis_begin = 0;
  pa.p_split = 0;
  pa.new_blk0 = 0;
  pa.group = group;
  pa.n_q_heads = n_q_heads;
  pa.q = static_cast<const uint16_t*>(q);
  pa.qscale = scale * 1.4426950408889634f;
  std::memcpy(pa.sign_bits, p->sign_bits, sizeof(pa.sign_bits));
  pa.c = p->c;
  pa.out = out;
  pa.out_f32 = out_dtype == FMKV_DTYPE_F32 ? 1 : 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  if (!stored) {
    e = fmkv::launch_append(ap, n_seqs, tasks, s);
    if (e != hipSuccess) return hip_fail(e, "paged append launch");
  }
  // (starts are on the device: the caller or the table's width bounds the lengths)
  int64_t blocks = ((int64_t)max_seq_len + fmkv::kBlockTokens - 1) / fmkv::kBlockTokens;
  if (blocks == 0 || blocks > max_blocks) blocks = max_blocks;
  // (a tile of 64 rows sees a window, its own positions and the sinks)
  if (window > 0) blocks = std::min(blocks, window_blocks((int64_t)window + 64, sinks));
  e = run_prefill(pa, p->split, p->cus, blocks / 2 + 2, s, window > 0 ? &p->ws : nullptr);
  if (e != hipSuccess) return hip_fail(e, "prefill attention launch");
  return FMKV_OK;
}

}  // namespace

extern "C" {

int fmkv_paged_prefill_step_bounded(fmkv_pool* p, const void* k, const void* v,
                                    const int32_t* block_tables, int32_t max_blocks,
                                    const int32_t* start_pos, int32_t n_seqs, int32_t n_new,
                                    int32_t max_seq_len, const void* q, int32_t n_q_heads,
                                    float scale, void* out, int32_t out_dtype, void* stream) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  return paged_prefill_impl(p, false, k, v, block_tables, max_blocks, start_pos, n_seqs, n_new,
                            max_seq_len, q, n_q_heads, scale, 0, 0, out, out_dtype, stream);
}

int fmkv_paged_window_prefill_step(fmkv_pool* p, const void* k, const void* v,
                                   const int32_t* block_tables, int32_t max_blocks,
                                   const int32_t* start_pos, int32_t n_seqs, int32_t n_new,
                                   int32_t max_seq_len, const void* q, int32_t n_q_heads,
                                   float scale, int32_t window, int32_t sinks, void* out,
                                   int32_t out_dtype, void* stream) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  const int rc = check_window(window, sinks);
  if (rc) return rc;
  return paged_prefill_impl(p, false, k, v, block_tables, max_blocks, start_pos, n_seqs, n_new,
                            max_seq_len, q, n_q_heads, scale, window, sinks, out, out_dtype, stream);
}

int fmkv_paged_window_prefill_attention(fmkv_pool* p, const void* q, const int32_t* block_tables,
                                        int32_t max_blocks, const int32_t* start_pos,
                                        int32_t n_seqs, int32_t n_new, int32_t max_seq_len,
                                        int32_t n_q_heads, float scale, int32_t window,
                                        int32_t sinks, void* out, int32_t out_dtype, void* stream) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  const int rc = check_window(window, sinks);
  if (rc) return rc;
  return paged_prefill_impl(p, true, nullptr, nullptr, block_tables, max_blocks, start_pos, n_seqs,
                            n_new, max_seq_len, q, n_q_heads, scale, window, sinks, out, out_dtype,
                            stream);
}

int fmkv_paged_window_decode_attention(fmkv_pool* p, const void* q, const int32_t* block_tables,
                                       int32_t max_blocks, const int32_t* seq_lens, int32_t n_seqs,
                                       int32_t max_seq_len, int32_t n_q_heads, float scale,
                                       int32_t window, int32_t sinks, void* out, int32_t out_dtype,
                                       void* stream) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  int rc = check_window(window, sinks);
  if (rc) return rc;
  if (!std::isfinite(scale)) return fail(FMKV_ERR_INVALID_ARG, "scale must be finite");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  fmkv::AttnArgs a;
  rc = prepare_paged_attention(p, q, block_tables, max_blocks, seq_lens, n_seqs, max_seq_len,
                               n_q_heads, scale, 0.0f, out, out_dtype, 0, s, &a, window, sinks);
  if (rc || n_seqs == 0) return rc;
  hipEvent_t e0, e1;
  next_events(&e0, &e1);
  hipError_t e = launch_attention(a, n_seqs, p->desc.n_kv_heads, s, e0, e1);
  if (e != hipSuccess) return hip_fail(e, "paged window attention launch");
  return FMKV_OK;
}

int fmkv_paged_append(fmkv_pool* p, const void* k, const void* v, const int32_t* block_tables,
                      int32_t max_blocks, const int32_t* start_pos, int32_t n_seqs, int32_t n_new,
                      void* stream) {
  fmkv::AppendArgs a;
  int tasks = 0;
  int rc = prepare_paged_append(p, k, v, block_tables, max_blocks, start_pos, n_seqs, n_new, &a,
                                &tasks);
  if (rc || n_seqs == 0 || n_new == 0) return rc;
  hipError_t e = fmkv::launch_append(a, n_seqs, tasks, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "paged append launch");
  return FMKV_OK;
}

int fmkv_paged_append_projected(fmkv_pool* p, const void* k, const void* v,
                                const int32_t* block_tables, int32_t max_blocks,
                                const int32_t* start_pos, int32_t n_seqs, int32_t n_new,
                                const fmkv_kv_prologue* pro, void* stream) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  int rc = check_prologue(p->desc, pro);
  if (rc) return rc;
  fmkv::AppendArgs a;
  int tasks = 0;
  rc = prepare_paged_append(p, k, pro->v_from_k ? k : v, block_tables, max_blocks, start_pos, n_seqs,
                            n_new, &a, &tasks);
  if (rc || n_seqs == 0 || n_new == 0) return rc;
  set_prologue(pro, &a);
  hipError_t e = fmkv::launch_append(a, n_seqs, tasks, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "paged append launch");
  return FMKV_OK;
}

int fmkv_paged_decode_attention(fmkv_pool* p, const void* q, const int32_t* block_tables,
                                int32_t max_blocks, const int32_t* seq_lens, int32_t n_seqs,
                                int32_t max_seq_len, int32_t n_q_heads, float scale, float tau,
                                void* out, int32_t out_dtype, void* stream) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  fmkv::AttnArgs a;
  int rc = prepare_paged_attention(p, q, block_tables, max_blocks, seq_lens, n_seqs, max_seq_len,
                                   n_q_heads, scale, tau, out, out_dtype, 0, s, &a);
  if (rc || n_seqs == 0) return rc;
  hipEvent_t e0, e1;
  next_events(&e0, &e1);
  hipError_t e = launch_attention(a, n_seqs, p->desc.n_kv_heads, s, e0, e1);
  if (e != hipSuccess) return hip_fail(e, "paged decode attention launch");
  return FMKV_OK;
}

}  // extern "C"

namespace {

int paged_decode_step_impl(fmkv_pool* p, const void* k, const void* v,
                           const int32_t* block_tables, int32_t max_blocks,
                           const int32_t* start_pos, const int32_t* seq_lens, int32_t n_seqs,
                           int32_t n_new, int32_t max_seq_len, const void* q, int32_t n_q_heads,
                           float scale, float tau, void* out, int32_t out_dtype, void* stream,
                           const fmkv_kv_prologue* pro, int32_t win = 0, int32_t sinks = 0) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  if (n_new < 1) return fail(FMKV_ERR_INVALID_ARG, "a decode step appends at least one token");
  int rc;
  if (pro && (rc = check_prologue(p->desc, pro))) return rc;
  fmkv::AppendArgs ap;
  int tasks = 0;
  rc = prepare_paged_append(p, k, pro && pro->v_from_k ? k : v, block_tables, max_blocks,
                            start_pos, n_seqs, n_new, &ap, &tasks);
  if (rc) return rc;
  if (pro) set_prologue(pro, &ap);
  // one new token per sequence: the attention launch appends it itself, at
  // position seq_lens[s] - 1 (= start_pos[s])
  const int fused = n_new == 1 ? 1 : 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  fmkv::AttnArgs at;
  rc = prepare_paged_attention(p, q, block_tables, max_blocks, seq_lens, n_seqs, max_seq_len,
                               n_q_heads, scale, tau, out, out_dtype, fused, s, &at, win, sinks);
  if (rc || n_seqs == 0) return rc;
  hipError_t e;
  if (fused) {
    at.k_new = ap.k;
    at.v_new = ap.v;
    if (pro) set_prologue(pro, &at);
  } else {
    e = fmkv::launch_append(ap, n_seqs, tasks, s);
    if (e != hipSuccess) return hip_fail(e, "paged append launch");
  }
  hipEvent_t e0, e1;
  next_events(&e0, &e1);
  e = launch_attention(at, n_seqs, p->desc.n_kv_heads, s, e0, e1);
  if (e != hipSuccess) return hip_fail(e, "paged decode attention launch");
  return FMKV_OK;
}

}  // namespace

extern "C" {

int fmkv_paged_decode_step(fmkv_pool* p, const void* k, const void* v,
                           const int32_t* block_tables, int32_t max_blocks,
                           const int32_t* start_pos, const int32_t* seq_lens, int32_t n_seqs,
                           int32_t n_new, int32_t max_seq_len, const void* q, int32_t n_q_heads,
                           float scale, float tau, void* out, int32_t out_dtype, void* stream) {
  return paged_decode_step_impl(p, k, v, block_tables, max_blocks, start_pos, seq_lens, n_seqs,
                                n_new, max_seq_len, q, n_q_heads, scale, tau, out, out_dtype,
                                stream, nullptr);
}

int fmkv_paged_window_decode_step(fmkv_pool* p, const void* k, const void* v,
                                  const int32_t* block_tables, int32_t max_blocks,
                                  const int32_t* start_pos, const int32_t* seq_lens,
                                  int32_t n_seqs, int32_t max_seq_len, const void* q,
                                  int32_t n_q_heads, float scale, int32_t window, int32_t sinks,
                                  void* out, int32_t out_dtype, void* stream) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  int rc = check_window(window, sinks);
  if (rc) return rc;
  if (!std::isfinite(scale)) return fail(FMKV_ERR_INVALID_ARG, "scale must be finite");
  return paged_decode_step_impl(p, k, v, block_tables, max_blocks, start_pos, seq_lens, n_seqs, 1,
                                max_seq_len, q, n_q_heads, scale, 0.0f, out, out_dtype, stream,
                                nullptr, window, sinks);
}

int fmkv_paged_decode_step_projected(fmkv_pool* p, const void* k_proj, const void* v_proj,
                                     const int32_t* block_tables, int32_t max_blocks,
                                     const int32_t* start_pos, const int32_t* seq_lens,
                                     int32_t n_seqs, int32_t n_new, int32_t max_seq_len,
                                     const fmkv_kv_prologue* pro, const void* q,
                                     int32_t n_q_heads, float scale, float tau, void* out,
                                     int32_t out_dtype, void* stream) {
  if (!pro) return fail(FMKV_ERR_INVALID_ARG, "prologue is null");
  return paged_decode_step_impl(p, k_proj, v_proj, block_tables, max_blocks, start_pos, seq_lens,
                                n_seqs, n_new, max_seq_len, q, n_q_heads, scale, tau, out,
                                out_dtype, stream, pro);
}

int fmkv_pools_copy_blocks(fmkv_pool* const* pools, int32_t n_pools, const int32_t* src,
                           const int32_t* dst, int64_t n_pairs, void* stream) {
  if (n_pools < 0 || n_pairs < 0) return fail(FMKV_ERR_INVALID_ARG, "n_pools and n_pairs must be >= 0");
  if (n_pools == 0 || n_pairs == 0) return FMKV_OK;
  if (!pools || !src || !dst) return fail(FMKV_ERR_INVALID_ARG, "pools/src/dst are null");
  for (int32_t i = 0; i < n_pools; i++)
    if (!pools[i]) return fail(FMKV_ERR_INVALID_ARG, "pool " + std::to_string(i) + " is null");
  for (int32_t i = 0; i < n_pools; i++) {
    const int rc = check_device(pools[i]);
    if (rc) return rc;
  }
  for (int32_t i0 = 0; i0 < n_pools; i0 += fmkv::kCopyPools) {
    fmkv::CopyArgs a;
    const int n = std::min<int32_t>(n_pools - i0, fmkv::kCopyPools);
    for (int i = 0; i < n; i++) {
      const fmkv_pool* p = pools[i0 + i];
      a.base[i] = p->arena;
      a.block_bytes[i] = p->layout.block_bytes * p->desc.n_kv_heads;
      a.n_blocks[i] = (int32_t)p->n_blocks;
    }
    a.src = src;
    a.dst = dst;
    const hipError_t e = fmkv::launch_copy_blocks(a, n, n_pairs, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "block copy launch");
  }
  return FMKV_OK;
}

int fmkv_paged_compact(fmkv_pool* p, const int32_t* block_tables, int32_t max_blocks,
                       const int32_t* keep, int32_t max_keep, const int32_t* n_keep,
                       const int32_t* dst_tables, int32_t dst_max_blocks, int32_t n_seqs,
                       void* stream) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  if (n_seqs < 0 || max_keep < 0 || max_blocks < 1 || dst_max_blocks < 1)
    return fail(FMKV_ERR_INVALID_ARG, "bad n_seqs / max_keep / max_blocks / dst_max_blocks");
  if (n_seqs > 65535) return fail(FMKV_ERR_INVALID_ARG, "at most 65535 sequences per call");
  if (n_seqs == 0 || max_keep == 0) return FMKV_OK;
  if (!block_tables || !keep || !n_keep || !dst_tables)
    return fail(FMKV_ERR_INVALID_ARG, "block_tables/keep/n_keep/dst_tables are null");
  // (a grid holds fewer than 2^32 threads in x, 256 a block)
  if (max_keep > (1 << 28) - 16) return fail(FMKV_ERR_INVALID_ARG, "max_keep must be <= 2^28 - 16");
  if (max_keep > (int64_t)dst_max_blocks * fmkv::kBlockTokens)
    return fail(FMKV_ERR_INVALID_ARG, "max_keep exceeds dst_max_blocks * 16");
  const int rc = check_device(p);
  if (rc) return rc;
  fmkv::CompactArgs a;
  a.st = pool_store(p, block_tables, max_blocks);
  a.dst_table = dst_tables;
  a.dst_stride = dst_max_blocks;
  a.keep = keep;
  a.max_keep = max_keep;
  a.n_keep = n_keep;
  const hipError_t e = fmkv::launch_compact(a, n_seqs, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "compact launch");
  return FMKV_OK;
}

int fmkv_qkv_norm_rope(const fmkv_qkv_prologue* pro, int32_t head_dim, int32_t n_q_heads,
                       int32_t n_kv_heads, int64_t n_tokens, const void* q, int64_t q_stride,
                       const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                       const int32_t* positions, void* q_out, void* k_out, void* v_out,
                       void* stream) {
  if (!pro) return fail(FMKV_ERR_INVALID_ARG, "prologue is null");
  if (head_dim != 128 && head_dim != 256 && head_dim != 512)
    return fail(FMKV_ERR_UNSUPPORTED, "head_dim must be 128, 256 or 512");
  if (n_q_heads < 0 || n_kv_heads < 0 || n_q_heads > 65535 || n_kv_heads > 65535 ||
      n_q_heads + n_kv_heads == 0)
    return fail(FMKV_ERR_INVALID_ARG, "n_q_heads and n_kv_heads must be in [0, 65535], one of them > 0");
  if (n_tokens < 0 || n_tokens > INT32_MAX) return fail(FMKV_ERR_INVALID_ARG, "n_tokens must be in [0, 2^31)");
  if (!(pro->eps > 0.0f) || !std::isfinite(pro->eps))
    return fail(FMKV_ERR_INVALID_ARG, "eps must be finite and > 0");
  if (!(pro->rope_theta >= 1.0f) || !std::isfinite(pro->rope_theta))
    return fail(FMKV_ERR_INVALID_ARG, "rope_theta must be finite and >= 1");
  if (pro->rope_dims < 0 || pro->rope_dims > head_dim || pro->rope_dims % 8 != 0)
    return fail(FMKV_ERR_UNSUPPORTED, "rope_dims must be a multiple of 8 in [0, head_dim]");
  if (pro->n_axes < 1 || pro->n_axes > 4) return fail(FMKV_ERR_INVALID_ARG, "n_axes must be 1 to 4");
  if ((pro->v_norm != 0 && pro->v_norm != 1) || (pro->v_from_k != 0 && pro->v_from_k != 1))
    return fail(FMKV_ERR_INVALID_ARG, "v_norm and v_from_k must be 0 or 1");
  fmkv::NormRopeArgs a;
  int64_t pairs = 0;
  for (int i = 0; i < 4; i++) {
    if (i < pro->n_axes && pro->n_axes > 1) {
      if (pro->sections[i] < 0) return fail(FMKV_ERR_INVALID_ARG, "sections must be >= 0");
      pairs += pro->sections[i];
    }
    // (pairs from the last axis's end on do not exist)
    a.axis_end[i] = i < pro->n_axes - 1 ? (int32_t)std::min<int64_t>(pairs, INT32_MAX) : INT32_MAX;
  }
  if (pro->n_axes > 1 && 2 * pairs != pro->rope_dims)
    return fail(FMKV_ERR_INVALID_ARG, "sections must add up to rope_dims / 2");
  const bool has_v = v != nullptr;
  if (pro->v_from_k && (has_v || n_kv_heads == 0))
    return fail(FMKV_ERR_INVALID_ARG, "v_from_k takes V from k: k rows and no v");
  const bool out_v = has_v || pro->v_from_k;
  // arguments of the rows that are there
  struct Rows {
    const char* name;
    bool there;
    const void* in;
    void* out;
    int64_t heads, stride;
    bool reads;
  } rows[3] = {{"q", n_q_heads > 0, q, q_out, n_q_heads, q_stride, true},
               {"k", n_kv_heads > 0, k, k_out, n_kv_heads, k_stride, true},
               {"v", n_kv_heads > 0 && out_v, v, v_out, n_kv_heads, v_stride, has_v}};
  for (const Rows& r : rows) {
    if (!r.there) {
      if (r.in) return fail(FMKV_ERR_INVALID_ARG, std::string(r.name) + " without heads");
      continue;
    }
    if ((r.reads && !r.in) || !r.out)
      return fail(FMKV_ERR_INVALID_ARG, std::string(r.name) + " and its output must be device pointers");
    if (r.reads && r.stride < r.heads * head_dim)
      return fail(FMKV_ERR_INVALID_ARG, std::string(r.name) + "_stride must be >= heads * head_dim");
    if (r.reads && r.stride > ((int64_t)1 << 31))
      return fail(FMKV_ERR_INVALID_ARG, std::string(r.name) + "_stride must be <= 2^31");
  }
  if ((n_q_heads > 0 && !pro->q_norm_weight) || (n_kv_heads > 0 && !pro->k_norm_weight))
    return fail(FMKV_ERR_INVALID_ARG, "norm weights must be device pointers");
  if (pro->rope_dims > 0 && !positions) return fail(FMKV_ERR_INVALID_ARG, "positions is null");
  if (n_tokens == 0) return FMKV_OK;
  // an output over an input or another output: rows would be read after they
  // were written (its own input, row for row, is read first)
  auto span = [&](const void* p, int64_t bytes) {
    return std::pair<uintptr_t, uintptr_t>((uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes);
  };
  // (nor over what every row reads: the weights and the positions)
  const struct {
    const char* name;
    const void* at;
    int64_t bytes;
  } shared[3] = {{"q_norm_weight", n_q_heads > 0 ? pro->q_norm_weight : nullptr, head_dim * 2},
                 {"k_norm_weight", n_kv_heads > 0 ? pro->k_norm_weight : nullptr, head_dim * 2},
                 {"positions", pro->rope_dims > 0 ? positions : nullptr, pro->n_axes * n_tokens * 4}};
  for (int i = 0; i < 3; i++) {
    if (!rows[i].there) continue;
    const auto o = span(rows[i].out, n_tokens * rows[i].heads * head_dim * 2);
    for (const auto& x : shared) {
      const auto in = span(x.at, x.bytes);
      if (x.at && o.first < in.second && in.first < o.second)
        return fail(FMKV_ERR_INVALID_ARG, std::string(rows[i].name) + "'s output overlaps " + x.name);
    }
    for (int j = 0; j < 3; j++) {
      if (!rows[j].there) continue;
      const auto in = span(rows[j].in, ((n_tokens - 1) * rows[j].stride + rows[j].heads * head_dim) * 2);
      const bool same = i == j && rows[i].in == rows[i].out && rows[i].stride == rows[i].heads * head_dim;
      if (rows[j].reads && !same && o.first < in.second && in.first < o.second)
        return fail(FMKV_ERR_INVALID_ARG, std::string(rows[i].name) + "'s output overlaps " + rows[j].name);
      const auto p = span(rows[j].out, n_tokens * rows[j].heads * head_dim * 2);
      if (j > i && o.first < p.second && p.first < o.second)
        return fail(FMKV_ERR_INVALID_ARG, std::string("the outputs of ") + rows[i].name + " and " +
                                              rows[j].name + " overlap");
    }
  }
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_out = static_cast<uint16_t*>(k_out);
  a.v_out = static_cast<uint16_t*>(v_out);
  a.q_w = static_cast<const uint16_t*>(pro->q_norm_weight);
  a.k_w = static_cast<const uint16_t*>(pro->k_norm_weight);
  a.pos = positions;
  a.n_tokens = n_tokens;
  a.n_q = n_q_heads;
  a.n_k = n_kv_heads;
  a.n_v = has_v ? n_kv_heads : 0;
  a.v_norm = pro->v_norm;
  a.v_from_k = pro->v_from_k;
  a.eps = pro->eps;
  a.rope_dims = pro->rope_dims;
  a.log2_theta = std::log2((double)pro->rope_theta);
  const hipError_t e =
      fmkv::launch_norm_rope(a, head_dim, device_cus(), static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "norm and rotation launch");
  return FMKV_OK;
}

int fmkv_pool_storage(const fmkv_pool* p, void** base, int64_t* block_bytes) {
  if (!p || !base || !block_bytes) return fail(FMKV_ERR_INVALID_ARG, "null argument");
  *base = p->arena;
  *block_bytes = p->layout.block_bytes * p->desc.n_kv_heads;
  return FMKV_OK;
}

int fmkv_pool_read_codes(const fmkv_pool* p, void* codes, void* meta, void* stream) {
  if (!p) return fail(FMKV_ERR_INVALID_ARG, "pool is null");
  if (!codes || (!meta && p->desc.mode != FMKV_MODE_PLAIN))
    return fail(FMKV_ERR_INVALID_ARG, "codes/meta must be device pointers");
  fmkv::ReadArgs a;
  a.st = pool_store(p, nullptr, 0);
  a.n_slots = p->n_blocks * fmkv::kBlockTokens;
  a.codes = static_cast<uint32_t*>(codes);
  a.meta = static_cast<uint16_t*>(meta);
  hipError_t e = fmkv::launch_read_codes(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "pool read_codes launch");
  return FMKV_OK;
}

int fmkv_set_sparse_v_gather(int32_t on) {
  if (on != 0 && on != 1) return fail(FMKV_ERR_INVALID_ARG, "sparse_v_gather must be 0 or 1");
  g_sparse_gather = on;
  return FMKV_OK;
}

int fmkv_set_blocks_per_split(int32_t bps) {
  if (bps < 0) return fail(FMKV_ERR_INVALID_ARG, "blocks_per_split must be >= 0");
  g_bps_override = bps;
  return FMKV_OK;
}

int fmkv_profile_enable(int32_t max_records) {
  if (max_records < 0 || max_records > (1 << 20))
    return fail(FMKV_ERR_INVALID_ARG, "max_records must be in [0, 2^20]");
  g_prof.clear_events();
  g_prof.max_records = 0;
  if (max_records == 0) return FMKV_OK;
  g_prof.ev.resize(2 * (size_t)max_records, nullptr);
  for (size_t i = 0; i < g_prof.ev.size(); i++) {
    hipError_t e = hipEventCreate(&g_prof.ev[i]);
    if (e != hipSuccess) {
      g_prof.ev.resize(i);
      g_prof.clear_events();
      return hip_fail(e, "hipEventCreate");
    }
  }
  g_prof.max_records = max_records;
  return FMKV_OK;
}

int fmkv_profile_collect(double* total_ms, int32_t* n_records) {
  if (!total_ms || !n_records) return fail(FMKV_ERR_INVALID_ARG, "null argument");
  double sum = 0.0;
  for (int32_t i = 0; i < g_prof.used; i++) {
    float ms;
    int rc = profile_pair_ms(i, &ms);
    if (rc) return rc;
    sum += ms;
  }
  *total_ms = sum;
  *n_records = g_prof.used;
  g_prof.used = 0;
  return FMKV_OK;
}

int fmkv_profile_collect_each(float* ms_out, int32_t capacity, int32_t* n_records) {
  if (!ms_out || !n_records) return fail(FMKV_ERR_INVALID_ARG, "null argument");
  if (capacity < g_prof.used)
    return fail(FMKV_ERR_CAPACITY, std::to_string(g_prof.used) + " records need a buffer of as "
                                   "many floats; capacity is " + std::to_string(capacity));
  for (int32_t i = 0; i < g_prof.used; i++) {
    int rc = profile_pair_ms(i, &ms_out[i]);
    if (rc) return rc;
  }
  *n_records = g_prof.used;
  g_prof.used = 0;
  return FMKV_OK;
}

}  // extern "C"

// ---------------------------------------------------------------------------
// The book of a pool's blocks (host only)
// ---------------------------------------------------------------------------

struct fmkv_pages {
  std::vector<int32_t> users;  // of each block
  std::vector<int32_t> free;   // blocks without users, the next one last
};

namespace {

int check_block(const fmkv_pages* p, int32_t block) {
  if (block < 0 || (size_t)block >= p->users.size())
    return fail(FMKV_ERR_INVALID_ARG, "block " + std::to_string(block) + " is not one of " +
                                          std::to_string(p->users.size()));
  if (p->users[block] == 0)
    return fail(FMKV_ERR_INVALID_ARG, "block " + std::to_string(block) + " is free");
  return FMKV_OK;
}

// A sequence's tokens: positions are 32-bit (start_pos, seq_lens).
int check_tokens(int64_t n_tokens) {
  if (n_tokens < 0 || n_tokens > INT32_MAX)
    return fail(FMKV_ERR_INVALID_ARG, "n_tokens must be in [0, 2^31)");
  return FMKV_OK;
}

}  // namespace

extern "C" {

int fmkv_pages_create(int64_t n_blocks, fmkv_pages** out) {
  if (!out) return fail(FMKV_ERR_INVALID_ARG, "out is null");
  *out = nullptr;
  if (n_blocks < 1 || n_blocks > ((int64_t)1 << 31) - 1)
    return fail(FMKV_ERR_INVALID_ARG, "n_blocks must be in [1, 2^31)");
  fmkv_pages* p = nullptr;
  try {
    p = new fmkv_pages();
    p->users.assign((size_t)n_blocks, 0);
    p->free.resize((size_t)n_blocks);
  } catch (const std::exception&) {
    delete p;
    return fail(FMKV_ERR_OOM, "no memory for the book of blocks");
  }
  for (int64_t i = 0; i < n_blocks; i++) p->free[i] = (int32_t)(n_blocks - 1 - i);
  *out = p;
  return FMKV_OK;
}

int fmkv_pages_destroy(fmkv_pages* p) {
  delete p;
  return FMKV_OK;
}

int fmkv_pages_free_count(const fmkv_pages* p, int64_t* out) {
  if (!p || !out) return fail(FMKV_ERR_INVALID_ARG, "null argument");
  *out = (int64_t)p->free.size();
  return FMKV_OK;
}

int fmkv_pages_users(const fmkv_pages* p, int32_t block, int32_t* out) {
  if (!p || !out) return fail(FMKV_ERR_INVALID_ARG, "null argument");
  if (block < 0 || (size_t)block >= p->users.size())
    return fail(FMKV_ERR_INVALID_ARG, "unknown block");
  *out = p->users[block];
  return FMKV_OK;
}

int fmkv_pages_alloc(fmkv_pages* p, int64_t n, int32_t* blocks) {
  if (!p || n < 0 || (n > 0 && !blocks)) return fail(FMKV_ERR_INVALID_ARG, "bad pages / n / blocks");
  if (n > (int64_t)p->free.size())
    return fail(FMKV_ERR_CAPACITY, std::to_string(n) + " blocks asked for, " +
                                       std::to_string(p->free.size()) + " free");
  for (int64_t i = 0; i < n; i++) {
    blocks[i] = p->free.back();
    p->free.pop_back();
    p->users[blocks[i]] = 1;
  }
  return FMKV_OK;
}

int fmkv_pages_release(fmkv_pages* p, const int32_t* blocks, int64_t n) {
  if (!p || n < 0 || (n > 0 && !blocks)) return fail(FMKV_ERR_INVALID_ARG, "bad pages / n / blocks");
  // (the free list has room for every block from the start: nothing is allocated)
  // The users first, so that a block listed more often than it is used is
  // noticed (and everything put back); then the free list
  for (int64_t i = 0; i < n; i++) {
    if (blocks[i] == -1) continue;
    const int rc = check_block(p, blocks[i]);
    if (rc) {
      while (i-- > 0)
        if (blocks[i] != -1) p->users[blocks[i]]++;
      return rc;
    }
    p->users[blocks[i]]--;
  }
  for (int64_t i = n; i-- > 0;) {  // (backwards: the first listed is the first taken again)
    if (blocks[i] == -1 || p->users[blocks[i]] != 0) continue;
    p->free.push_back(blocks[i]);
    p->users[blocks[i]] = -1;  // listed once, whatever its users were
  }
  for (int64_t i = 0; i < n; i++)
    if (blocks[i] != -1 && p->users[blocks[i]] == -1) p->users[blocks[i]] = 0;
  return FMKV_OK;
}

int fmkv_pages_fork(fmkv_pages* p, const int32_t* blocks, int64_t n_tokens, int32_t* child,
                    int32_t* copy_src, int32_t* copy_dst) {
  if (int rc = check_tokens(n_tokens)) return rc;
  if (!p || !copy_src || !copy_dst || (n_tokens > 0 && (!blocks || !child)))
    return fail(FMKV_ERR_INVALID_ARG, "pages/blocks/child/copy_src/copy_dst are null");
  const int64_t n = (n_tokens + fmkv::kBlockTokens - 1) / fmkv::kBlockTokens;
  const bool part = n_tokens % fmkv::kBlockTokens != 0;
  if (part && blocks[n - 1] == -1)
    return fail(FMKV_ERR_INVALID_ARG, "the block that the sequence would go on in was given back");
  for (int64_t i = 0; i < n; i++) {
    if (blocks[i] == -1) continue;
    const int rc = check_block(p, blocks[i]);
    if (rc) return rc;
    if (p->users[blocks[i]] == INT32_MAX) return fail(FMKV_ERR_CAPACITY, "a block has 2^31 - 1 users");
  }
  int32_t fresh = -1;
  if (part) {
    const int rc = fmkv_pages_alloc(p, 1, &fresh);
    if (rc) return rc;
  }
  *copy_src = part ? blocks[n - 1] : -1;
  *copy_dst = fresh;
  for (int64_t i = 0; i < n; i++) {
    const bool copied = part && i == n - 1;
    if (blocks[i] != -1 && !copied) p->users[blocks[i]]++;
    child[i] = copied ? fresh : blocks[i];
  }
  return FMKV_OK;
}

int fmkv_pages_slide(fmkv_pages* p, int32_t* blocks, int64_t n_tokens, int32_t window,
                     int32_t sinks, int64_t* n_freed) {
  int rc = check_tokens(n_tokens);
  if (rc) return rc;
  if (!p || (n_tokens > 0 && !blocks) || !n_freed)
    return fail(FMKV_ERR_INVALID_ARG, "pages/blocks/n_freed are null");
  if ((rc = check_window(window, sinks))) return rc;
  constexpr int64_t B = fmkv::kBlockTokens;
  // blocks [first, last) hold hidden positions alone: from the sinks' end to the
  // window of the next query, at position n_tokens
  const int64_t first = ((int64_t)sinks + B - 1) / B, last = std::max<int64_t>(n_tokens + 1 - window, 0) / B;
  *n_freed = 0;
  if (last <= first) return FMKV_OK;
  if ((rc = fmkv_pages_release(p, blocks + first, last - first))) return rc;
  for (int64_t i = first; i < last; i++) {
    *n_freed += blocks[i] != -1;
    blocks[i] = -1;
  }
  return FMKV_OK;
}

}  // extern "C"
