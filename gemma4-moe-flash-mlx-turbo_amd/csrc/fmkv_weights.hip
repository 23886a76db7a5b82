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
constexpr int kKeepCopies = 16;  // of the histogram, by lane

// Weights as unsigned numbers of the same order, equal for equal weights (both
// zeros are one); a NaN is below every weight.
__device__ inline uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One work-group per sequence. Of T > max_keep positions the first `sinks` and the
// last `recent` stay, and as many of the others, the heaviest, as make max_keep:
// the B-th largest key digit by digit (8 bits, from the top: a histogram of the
// keys that share the digits found so far), then every larger one and the first of
// the equal ones, written in the order of the positions.
__global__ __launch_bounds__(kKeepThreads) void heaviest_kernel(HeaviestArgs a) {
  __shared__ uint32_t hist[256 * kKeepCopies];
  __shared__ uint32_t counts[256];
  __shared__ uint32_t found[2];  // the digit, keys above it
  __shared__ int wave_above[kKeepWaves], wave_equal[kKeepWaves];
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t T = a.seq_lens[seq];
  T = T < 0 ? 0 : T > a.width ? a.width : T;
  const float* w = a.weights + (int64_t)seq * a.width;
  int32_t* keep = a.keep + (int64_t)seq * a.max_keep;
  float* kept = a.kept ? a.kept + (int64_t)seq * a.kept_width : nullptr;
  const int n = (int)(T < a.max_keep ? T : a.max_keep);
  if (tid == 0) a.n_keep[seq] = n;
  if (kept)
    for (int64_t i = n + tid; i < a.kept_width; i += kKeepThreads) kept[i] = 0.0f;
  auto put = [&](int at, int64_t i) {
    keep[at] = (int32_t)i;
    if (kept) kept[at] = w[i];
  };
  if (T <= a.max_keep) {
    for (int64_t i = tid; i < T; i += kKeepThreads) put((int)i, i);
    return;
  }
  const int64_t lo = a.sinks, hi = T - a.recent;  // the positions between
  for (int i = tid; i < a.sinks; i += kKeepThreads) put(i, i);
  for (int i = tid; i < a.recent; i += kKeepThreads) put(n - a.recent + i, hi + i);
  uint32_t need = (uint32_t)(n - a.sinks - a.recent);
  if (need == 0) return;

  uint32_t prefix = 0, mask = 0;  // the digits found
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256 * kKeepCopies; i += kKeepThreads) hist[i] = 0;
    __syncthreads();
    for (int64_t i = lo + tid; i < hi; i += kKeepThreads) {
      const uint32_t k = weight_key(w[i]);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift & 255u) * kKeepCopies + (lane & (kKeepCopies - 1))], 1u);
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t c = 0;
      for (int i = 0; i < kKeepCopies; i++) c += hist[tid * kKeepCopies + ((tid + i) & (kKeepCopies - 1))];
      counts[tid] = c;
    }
    __syncthreads();
    if (wave == 0) {  // lane l: digits 255 - 4 l .. 252 - 4 l
      uint32_t c[4], sum = 0;
      for (int i = 0; i < 4; i++) c[i] = counts[255 - 4 * lane - i], sum += c[i];
      uint32_t upto = sum;  // keys of the lanes 0 .. l
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)upto, d);
        if (lane >= d) upto += o;
      }
      uint32_t above = upto - sum;
      for (int i = 0; i < 4; i++) {
        if (above < need && above + c[i] >= need) found[0] = 255 - 4 * lane - i, found[1] = above;
        above += c[i];
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= 255u << shift;
    need -= found[1];
    __syncthreads();
  }
  // `need` of the keys equal to prefix, the first ones, and all above it. A
  // wave takes a run of positions; what the waves before it keep gives its place.
  const int64_t run = (hi - lo + kKeepWaves - 1) / kKeepWaves;
  const int64_t r0 = lo + wave * run < hi ? lo + wave * run : hi, r1 = r0 + run < hi ? r0 + run : hi;
  int above = 0, equal = 0;
  for (int64_t i = r0 + lane; i < r1; i += 64) {
    const uint32_t k = weight_key(w[i]);
    above += k > prefix;
    equal += k == prefix;
  }
  for (int d = 1; d < 64; d <<= 1) above += __shfl_xor(above, d), equal += __shfl_xor(equal, d);
  if (lane == 0) wave_above[wave] = above, wave_equal[wave] = equal;
  __syncthreads();
  above = equal = 0;
  for (int i = 0; i < wave; i++) above += wave_above[i], equal += wave_equal[i];
  int equal_left = (int)need - equal;  // of this wave's equal keys
  int at = a.sinks + above + (equal < (int)need ? equal : (int)need);
  for (int64_t i0 = r0; i0 < r1; i0 += 64) {
    const int64_t i = i0 + lane;
    const uint32_t k = i < r1 ? weight_key(w[i]) : 0u;
    const bool eq = i < r1 && k == prefix;
    const uint64_t below = (1ull << lane) - 1ull;
    const uint64_t eqs = __ballot(eq);
    const bool take = i < r1 && (k > prefix || (eq && (int)__popcll(eqs & below) < equal_left));
    const uint64_t takes = __ballot(take);
    if (take) put(at + (int)__popcll(takes & below), i);
    at += (int)__popcll(takes);
    equal_left -= (int)__popcll(eqs);
  }
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
