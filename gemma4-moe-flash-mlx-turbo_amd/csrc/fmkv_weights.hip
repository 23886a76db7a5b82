// Accumulated attention weights: how much each position of a cache has been
// attended to, and the positions that an eviction by it keeps.
//
// weight[s][j] is the sum, over query heads h (and over the steps or queries that
// are accumulated), of p_h(j) = 2^(s_h(j) - M_h) / L_h, s_h the base-2 scores of a
// softmax, M_h and L_h its maximum and sum. A decode step's split kernels store
// their scores; what they cannot know, M and L over all splits, this launch takes
// from the partials that it merges for the output anyway.
#include "fmkv_device.h"
#include "fmkv_internal.h"
#include "fmkv_combine.h"

namespace fmkv {
namespace {

constexpr int kWeighThreads = 256;  // positions of a work-group
constexpr int kWeighHeads = 64;     // query heads whose M and 1 / L are held at a time

// The split merge, and the weights: grid x counts the merge's work-groups (64
// dims, q head, sequence), then n_parts of 256 positions for each sequence. A position is
// one thread's, which adds its heads up in order: no atomics, the same sum each time.
// (32 sequences of 512 .. 16384 positions, 16 heads of 256 dims: 10.2 us, where the merge alone
// takes 5; the stores of the scores cost the split kernel 10 us of its 100.)
template <int D>
__global__ __launch_bounds__(kWeighThreads) void combine_weigh_kernel(AttnArgs a, uint32_t flags,
                                                                      int n_seqs, int n_parts) {
  const uint32_t merges = (uint32_t)(D / 64) * a.n_q_heads * n_seqs;
  if (blockIdx.x < merges) {
    const uint32_t row = blockIdx.x / (D / 64), seq = row / (uint32_t)a.n_q_heads;
    combine_rows<D>(a.part_o, a.part_ml, a.out, -1, a.part_stride, flags, a, blockIdx.x % (D / 64),
                    row - seq * a.n_q_heads, seq, n_seqs);
    return;
  }
  __shared__ float2 stat[kWeighHeads];  // M, 1 / L
  const int tid = threadIdx.x, lane = tid & 63;
  const uint32_t w = blockIdx.x - merges;
  const int seq = (int)(w / (uint32_t)n_parts);
  const int64_t T = a.seq_lens[seq];
  const int64_t first = (int64_t)(w - (uint32_t)seq * n_parts) * kWeighThreads;
  const int64_t end = T < a.weights_width ? T : a.weights_width;
  if (first >= end) return;
  const int64_t p = first + tid;
  const int Hq = a.n_q_heads;
  const int n_splits = n_splits_for(attn_window(a, seq, T).geo, a.bps0, a.bps, a.max_splits, a.skew_p);
  const float* ml = a.part_ml + (int64_t)seq * a.part_stride * Hq * 2;
  // positions whose scores are stored (the new token's comes from its column's partial)
  const int64_t blk = p / kBlockTokens;
  const bool stored = p < end && blk < a.score_blocks && blk < a.st.table_stride;
  const bool fresh = a.new_col && p == T - 1;
  const float* sc = a.scores + ((int64_t)seq * a.score_blocks + (stored ? blk : 0)) * Hq * kBlockTokens +
                    (p & (kBlockTokens - 1));
  float sum = 0.0f;
  for (int h0 = 0; h0 < Hq; h0 += kWeighHeads) {
    const int nh = Hq - h0 < kWeighHeads ? Hq - h0 : kWeighHeads;
    // sixteen lanes a head: each merges every sixteenth split, then they meet
    for (int h = tid >> 4; h < nh; h += kWeighThreads / 16) {
      float M = -1e30f, L = 0.0f;
      for (int s = tid & 15; s < n_splits + a.new_col; s += 16) {
        const float2 x = *reinterpret_cast<const float2*>(ml + ((int64_t)s * Hq + h0 + h) * 2);
        const float mn = fmaxf(M, x.x);
        L = fmaf(L, exp2f(M - mn), x.y * exp2f(x.x - mn));
        M = mn;
      }
      const float Mx = group_max<16>(M, lane);
      L = group_sum<16>(L * exp2f(M - Mx), lane);
      if ((tid & 15) == 0) stat[h] = make_float2(Mx, L > 0.0f ? 1.0f / L : 0.0f);
    }
    __syncthreads();
    if (stored) {
#pragma unroll 8
      for (int h = 0; h < nh; h++) {
        const float2 z = stat[h];
        sum = fmaf(exp2f(sc[(int64_t)(h0 + h) * kBlockTokens] - z.x), z.y, sum);
      }
    }
    if (fresh) {
      for (int h = 0; h < nh; h++)
        sum = fmaf(exp2f(ml[((int64_t)n_splits * Hq + h0 + h) * 2] - stat[h].x), stat[h].y, sum);
    }
    __syncthreads();
  }
  if (p < end) {
    const int64_t at = (int64_t)seq * a.weights_width + p;
    a.weights_out[at] = (a.weights_in ? a.weights_in[at] : 0.0f) + sum;
  }
}

// ---------------------------------------------------------------------------
// The positions that are kept
// ---------------------------------------------------------------------------

constexpr int kKeepThreads = 1024;
constexpr int kKeepWaves = kKeepThreads / 64;
constexpr int kKeepDigit = 12, kKeepBins = 1 << kKeepDigit;  // the first digit of a key
constexpr int kKeepLast = (32 - kKeepDigit) / 2;             // the other two
constexpr int kKeepRanked = 256;  // keys that one wave parts, four a lane

// Weights as unsigned numbers of the same order, equal for equal weights (both
// zeros are one); a NaN is below every weight.
__device__ inline uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct KeepShared {
  uint32_t hist[kKeepBins];
  uint32_t key[kKeepRanked], at[kKeepRanked];  // of a bin: keys, positions
  uint32_t sum[3][kKeepWaves];
  uint32_t bin, above, count, n_ranked;
  uint32_t last_key, last_at;  // of the positions that are kept, the last in order of (weight, position)
};

// Sums of the waves before this one; every thread calls it (one barrier).
__device__ inline uint32_t waves_before(uint32_t mine, uint32_t* sum, int wave, int lane) {
  if (lane == 0) sum[wave] = mine;
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < kKeepWaves; w++) before += w < wave ? sum[w] : 0u;
  return before;
}

// One wave, `count` keys and positions of sh that share the key's bits above `bits`, the
// positions below n: the need-th in order of falling key, then rising position. The bits
// of it are found from the top, each by how many of the keys left have it set. (Sixteen keys
// a lane instead of another digit of all keys took 10 us of 16384.)
__device__ inline void part_bin(KeepShared& sh, uint32_t count, uint32_t need, int bits, int64_t n, int lane) {
  constexpr int V = kKeepRanked / 64;
  uint32_t key[V], at[V], left = 0;  // bit v: the lane's v-th is left
#pragma unroll
  for (int v = 0; v < V; v++) {
    const uint32_t e = v * 64 + lane;
    const bool in = e < count;
    key[v] = in ? sh.key[e] : 0u;
    at[v] = in ? ~sh.at[e] : 0u;  // (the larger the earlier)
    left |= (uint32_t)in << v;
  }
  uint32_t n_left = count;
  auto part = [&](const uint32_t (&x)[V], int from) {
#pragma unroll 1
    for (int bit = from; bit >= 0 && n_left > need; bit--) {
      uint32_t set = 0;
      uint32_t n = 0;
#pragma unroll
      for (int v = 0; v < V; v++) {
        const bool b = (left >> v & 1u) && (x[v] >> bit & 1u);
        set |= (uint32_t)b << v;
        n += (uint32_t)__popcll(__ballot(b));
      }
      if (n >= need) {
        left = set;
        n_left = n;
      } else {
        need -= n;
        left &= ~set;
        n_left -= n;
      }
    }
  };
  part(key, bits - 1);
  part(at, 31 - __builtin_clz((uint32_t)n));  // (higher bits are all alike)
  // all that are left are kept: the least of them in that order
  uint32_t k = 0xffffffffu, a = 0;
#pragma unroll
  for (int v = 0; v < V; v++)
    if (left >> v & 1u) {
      const uint32_t p = ~at[v];
      if (key[v] < k || (key[v] == k && p > a)) k = key[v], a = p;
    }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t ok = (uint32_t)__shfl_xor((int)k, d), oa = (uint32_t)__shfl_xor((int)a, d);
    if (ok < k || (ok == k && oa > a)) k = ok, a = oa;
  }
  if (lane == 0) sh.last_key = k, sh.last_at = a;
}

// Of the n weights w[0 .. n) the heaviest `need` (0 < need < n), equal ones in
// order of position, to put(rank in order of position, position, weight). A wave
// takes a run of positions, a lane every 64th of it: KPT of them at most, in
// registers (0: any number, read again whenever they are looked at).
//   1. The need-th largest key's first 12 bits, from a histogram of all keys' (the
//      next 10 and the last 10 where the bin still holds more than a wave parts).
//   2. One wave finds the last one kept among the keys of that bin (part_bin).
//   3. Each wave writes its own, behind those of the waves before it.
template <int KPT, class Put>
__device__ inline void keep_heaviest(const float* w, int64_t n, uint32_t need, KeepShared& sh, Put put) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t run = (n + kKeepThreads - 1) / kKeepThreads * 64, r0 = wave * run + lane;
  const int kpt = (int)(run / 64);
  const uint64_t below = (1ull << lane) - 1ull;
  float held[KPT ? KPT : 1];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int t = 0; t < KPT; t++) {
      const int64_t i = r0 + t * 64;
      held[t] = t < kpt && i < n ? w[i] : 0.0f;
    }
  }
  // f(weight, position, there is one) of the thread's positions
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (KPT > 0) {
#pragma unroll
      for (int t = 0; t < KPT; t++) {
        const int64_t i = r0 + t * 64;
        if (t < kpt) f(held[t], i, i < n);  // (uniform)
      }
    } else {
      for (int t = 0; t < kpt; t++) {
        const int64_t i = r0 + (int64_t)t * 64;
        f(i < n ? w[i] : 0.0f, i, i < n);
      }
    }
  };
  uint32_t prefix = 0, mask = 0, count = 0;
  int shift = 32 - kKeepDigit;
#pragma unroll 1
  for (int digit = 0;; digit++) {
    const uint32_t bins = digit == 0 ? kKeepBins : 1u << kKeepLast;
#pragma unroll
    for (int i = 0; i < kKeepBins / kKeepThreads; i++) sh.hist[i * kKeepThreads + tid] = 0;
    __syncthreads();
    each([&](float x, int64_t, bool in) {
      const uint32_t k = weight_key(x);
      if (in && (k & mask) == prefix) atomicAdd(&sh.hist[k >> shift & (bins - 1u)], 1u);
    });
    __syncthreads();
    // thread t: four bins from 4095 - 4 t down, the heaviest first
    constexpr int kPer = kKeepBins / kKeepThreads;
    uint32_t c[kPer], sum = 0;
    const int top = kKeepBins - 1 - kPer * tid;
#pragma unroll
    for (int i = 0; i < kPer; i++) c[i] = sh.hist[top - i], sum += c[i];
    const uint32_t upto = (uint32_t)scan_add((int)sum);
    uint32_t above =
        waves_before((uint32_t)__builtin_amdgcn_readlane((int)upto, 63), sh.sum[0], wave, lane) + upto - sum;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (above < need && above + c[i] >= need) sh.bin = top - i, sh.above = above, sh.count = c[i];
      above += c[i];
    }
    if (tid == 0) sh.n_ranked = 0;
    __syncthreads();
    prefix |= sh.bin << shift;
    mask |= (bins - 1u) << shift;
    need -= sh.above;
    count = sh.count;
    if (count <= kKeepRanked || shift == 0) break;
    shift -= kKeepLast;
  }
  if (count <= kKeepRanked) {
    each([&](float x, int64_t i, bool in) {
      const uint32_t k = weight_key(x);
      const bool mine = in && (k & mask) == prefix;
      const uint64_t m = __ballot(mine);
      if (m) {
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&sh.n_ranked, (uint32_t)__popcll(m));
        at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + (uint32_t)__popcll(m & below);
        if (mine) sh.key[at] = k, sh.at[at] = (uint32_t)i;
      }
    });
    __syncthreads();
    if (wave == 0) part_bin(sh, count, need, shift, n, lane);
  } else {  // more equal keys than a wave parts: the need-th of them in order
    uint32_t equal = 0;
    each([&](float x, int64_t, bool in) { equal += (uint32_t)__popcll(__ballot(in && weight_key(x) == prefix)); });
    uint32_t before = waves_before(equal, sh.sum[1], wave, lane);
    each([&](float x, int64_t i, bool in) {
      const bool eq = in && weight_key(x) == prefix;
      const uint64_t m = __ballot(eq);
      if (eq && before + (uint32_t)__popcll(m & below) == need - 1u) sh.last_key = prefix, sh.last_at = (uint32_t)i;
      before += (uint32_t)__popcll(m);
    });
  }
  __syncthreads();
  const uint32_t last_key = sh.last_key, last_at = sh.last_at;
  auto taken = [&](float x, int64_t i, bool in) __attribute__((always_inline)) {
    const uint32_t k = weight_key(x);
    return in && (k > last_key || (k == last_key && (uint32_t)i <= last_at));
  };
  uint32_t mine = 0;
  each([&](float x, int64_t i, bool in) { mine += (uint32_t)__popcll(__ballot(taken(x, i, in))); });
  uint32_t at = waves_before(mine, sh.sum[2], wave, lane);
  each([&](float x, int64_t i, bool in) {
    const bool take = taken(x, i, in);
    const uint64_t m = __ballot(take);
    if (take) put((int)(at + (uint32_t)__popcll(m & below)), i, x);
    at += (uint32_t)__popcll(m);
  });
}

// One work-group per sequence: bound by its chain of loads, histogram, parting and
// barriers (one of 5003 positions 8.8 us, 32 of 512 .. 16384 15.2). Of T > max_keep positions the first `sinks` and the
// last `recent` stay, and as many of the others, the heaviest, as make max_keep.
__global__ __launch_bounds__(kKeepThreads) void heaviest_kernel(HeaviestArgs a) {
  __shared__ KeepShared sh;
  const int seq = blockIdx.x, tid = threadIdx.x;
  int64_t T = a.seq_lens[seq];
  T = T < 0 ? 0 : T > a.width ? a.width : T;
  const float* w = a.weights + (int64_t)seq * a.width;
  int32_t* keep = a.keep + (int64_t)seq * a.max_keep;
  float* kept = a.kept ? a.kept + (int64_t)seq * a.kept_width : nullptr;
  const int n = (int)(T < a.max_keep ? T : a.max_keep);
  if (tid == 0) a.n_keep[seq] = n;
  if (kept)
    for (int64_t i = n + tid; i < a.kept_width; i += kKeepThreads) kept[i] = 0.0f;
  auto put = [&](int at, int64_t i, float x) __attribute__((always_inline)) {
    keep[at] = (int32_t)i;
    if (kept) kept[at] = x;
  };
  // positions first .. first + count - 1 to places at ..
  auto put_run = [&](int at, int64_t first, int count) __attribute__((always_inline)) {
#pragma unroll 4
    for (int i = tid; i < count; i += kKeepThreads) put(at + i, first + i, w[first + i]);
  };
  if (T <= a.max_keep) {
    put_run(0, 0, n);
    return;
  }
  const int64_t lo = a.sinks, hi = T - a.recent;  // the positions between
  put_run(0, 0, a.sinks);
  put_run(n - a.recent, hi, a.recent);
  const uint32_t need = (uint32_t)(n - a.sinks - a.recent);
  if (need == 0) return;
  auto put_mid = [&](int at, int64_t i, float x) __attribute__((always_inline)) { put(a.sinks + at, lo + i, x); };
  if (hi - lo <= 8 * kKeepThreads)
    keep_heaviest<8>(w + lo, hi - lo, need, sh, put_mid);
  else if (hi - lo <= 16 * kKeepThreads)
    keep_heaviest<16>(w + lo, hi - lo, need, sh, put_mid);
  else
    keep_heaviest<0>(w + lo, hi - lo, need, sh, put_mid);
}

}  // namespace

hipError_t launch_combine_weigh(const AttnArgs& a, int n_seqs, hipStream_t s) {
  if (!a.seq_lens || a.n_q_heads >= (1 << 24) || a.tau > 0.0f) return hipErrorInvalidValue;
  const int D = a.st.layout.head_dim;
  const int n_parts = (int)((a.score_blocks * kBlockTokens + kWeighThreads - 1) / kWeighThreads);
  const int64_t grid = ((int64_t)(D / 64) * a.n_q_heads + n_parts) * n_seqs;
  if (grid * kWeighThreads > UINT32_MAX) return hipErrorInvalidValue;
  const uint32_t flags = (a.out_f32 ? 1u : 0u) | ((uint32_t)a.n_q_heads << 8);
  const auto kernel = D == 128   ? combine_weigh_kernel<128>
                      : D == 256 ? combine_weigh_kernel<256>
                                 : combine_weigh_kernel<512>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kWeighThreads), 0, s, a, flags, n_seqs, n_parts);
  return hipGetLastError();
}

hipError_t launch_heaviest(const HeaviestArgs& a, int n_seqs, hipStream_t s) {
  hipLaunchKernelGGL(heaviest_kernel, dim3(n_seqs), dim3(kKeepThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace fmkv
