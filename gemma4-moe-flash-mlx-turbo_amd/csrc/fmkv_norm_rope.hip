// Norms of q, k and v for each head and the rotation of q and k by their
// positions, in one pass over the projected rows.
//
//   y = x / sqrt(sum x^2 / D + eps) * w          (v: no w)
//   (y_i, y_{i + r/2}) <- (y_i c - y_{i+r/2} s, y_{i+r/2} c + y_i s),  i < r/2,
// c and s of the angle pos[axis(i)] * theta^(-2i/r), r = rope_dims; all in 32
// bits, rounded once to bf16 at the end.
//
// Bound by memory: every row is read once and written once. A row is taken by
// D / 8 lanes (a wave holds 4, 2 or 1 rows), each with both halves of four pairs
// (or eight unrotated dims), so that no lane needs another's values; only the
// sum of squares crosses lanes. A lane's sines and cosines are those of its four
// pairs, computed once per token and used for every head of it.
//
// 8192 tokens of 16 q, 2 k and 2 v rows of 512 dims, 128 of them rotated: 70 us for
// 336 MB, 4.8 TB/s; 32 tokens of 32 rows of 256 dims: 3.9 us in a graph.
//
// Angles: the frequency in turns, theta^(-2i/r) / 2 pi, is held as a fraction
// of 2^64; times the position modulo 2^64 it is the angle's fraction of a turn
// to 2^-24 at any 32-bit position, where an angle in 32 bits loses all but a
// few bits (position 10^5: 2^-7). The sines take the fraction in turns.
#include <cmath>

#include "fmkv_device.h"
#include "fmkv_internal.h"

namespace fmkv {
namespace {

constexpr int kNrThreads = 256;
constexpr int kNrAhead = 2;  // row groups of a wave whose loads are in flight together

// Four consecutive bf16 at an address aligned to one of them.
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef u16x4 u16x4_a2 __attribute__((aligned(2)));

__device__ inline void widen(u16x4 w, float* x) {
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = bf16_to_f32(w[i]);
}

template <int D>
__global__ __launch_bounds__(kNrThreads) void norm_rope_kernel(NormRopeArgs a) {
  constexpr int LPR = D / 8, RPW = 64 / LPR;  // lanes per row, rows per wave
  __shared__ uint64_t s_freq[D / 2];
  const int tid = threadIdx.x, lane = tid & 63, l = lane & (LPR - 1), sub = lane / LPR;
  const int half = a.rope_dims / 2;
  if (tid < half) {
    double f = exp2(-(double)tid / half * a.log2_theta) * 0.15915494309189535;  // / 2 pi
    s_freq[tid] = (uint64_t)(f * 18446744073709551616.0);
  }
  // The lane's dims da .. da + 3 and db .. db + 3: four pairs, or (past the
  // rotated ones) four of either half of the rest, so that a wave's loads and
  // stores are whole lines. (Eight in a row: two accesses to every line.)
  const bool rot = l < half / 4;
  const int da = rot ? 4 * l : a.rope_dims + 4 * (l - half / 4);
  const int db = da + (rot ? half : D / 2 - half);
  float qw[8], kw[8];
  if (a.n_q) {
    widen(*reinterpret_cast<const u16x4_a2*>(a.q_w + da), qw);
    widen(*reinterpret_cast<const u16x4_a2*>(a.q_w + db), qw + 4);
  }
  if (a.n_k) {
    widen(*reinterpret_cast<const u16x4_a2*>(a.k_w + da), kw);
    widen(*reinterpret_cast<const u16x4_a2*>(a.k_w + db), kw + 4);
  }
  __syncthreads();
  uint64_t freq[4];
  int axis[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    freq[i] = rot ? s_freq[da + i] : 0;
    axis[i] = (da + i >= a.axis_end[0]) + (da + i >= a.axis_end[1]) + (da + i >= a.axis_end[2]);
  }

  const int rows = a.n_q + a.n_k + a.n_v, groups = (rows + RPW - 1) / RPW;
  const int per = (groups + a.chunks - 1) / a.chunks;
  const int64_t tasks = a.n_tokens * a.chunks;
  const int64_t waves = (int64_t)gridDim.x * (kNrThreads / 64);
  for (int64_t task = (int64_t)blockIdx.x * (kNrThreads / 64) + (tid >> 6); task < tasks; task += waves) {
    const int64_t t = task / a.chunks;
    const int g0 = (int)(task - t * a.chunks) * per, g1 = g0 + per < groups ? g0 + per : groups;
    float cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t p = rot ? (int64_t)a.pos[axis[i] * a.n_tokens + t] : 0;
      // the fraction of a turn, as a signed 32-bit one
      const float turns = (float)(int32_t)((freq[i] * (uint64_t)p) >> 32) * 0x1p-32f;
      cs[i] = __builtin_amdgcn_cosf(turns);
      sn[i] = __builtin_amdgcn_sinf(turns);
    }
    for (int g = g0; g < g1; g += kNrAhead) {
      u16x4 wa[kNrAhead], wb[kNrAhead];
#pragma unroll
      for (int u = 0; u < kNrAhead; u++) {
        const int r = (g + u) * RPW + sub;
        if (g + u < g1 && r < rows) {
          const uint16_t* src = r < a.n_q           ? a.q + t * a.q_stride + (int64_t)r * D
                                : r < a.n_q + a.n_k ? a.k + t * a.k_stride + (int64_t)(r - a.n_q) * D
                                                    : a.v + t * a.v_stride + (int64_t)(r - a.n_q - a.n_k) * D;
          wa[u] = *reinterpret_cast<const u16x4_a2*>(src + da);
          wb[u] = *reinterpret_cast<const u16x4_a2*>(src + db);
        } else {
          wa[u] = wb[u] = (u16x4){0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int u = 0; u < kNrAhead; u++) {
        const int r = (g + u) * RPW + sub;
        float x[8];
        widen(wa[u], x);
        widen(wb[u], x + 4);
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
        ss = group_sum<LPR>(ss, lane);
        const float rn = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
        if (g + u >= g1 || r >= rows) continue;
        const bool isq = r < a.n_q, isk = !isq && r < a.n_q + a.n_k;
        if (isq || isk) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; i++) y[i] = x[i] * rn * (isq ? qw[i] : kw[i]);
          if (rot) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float ya = y[i], yb = y[i + 4];
              y[i] = fmaf(ya, cs[i], -yb * sn[i]);
              y[i + 4] = fmaf(yb, cs[i], ya * sn[i]);
            }
          }
          uint16_t* dst = isq ? a.q_out + (t * a.n_q + r) * D : a.k_out + (t * a.n_k + r - a.n_q) * D;
          u16x4 oa, ob;
#pragma unroll
          for (int i = 0; i < 4; i++) oa[i] = f32_to_bf16(y[i]), ob[i] = f32_to_bf16(y[i + 4]);
          *reinterpret_cast<u16x4_a2*>(dst + da) = oa;
          *reinterpret_cast<u16x4_a2*>(dst + db) = ob;
        }
        if (isk ? a.v_from_k : !isq) {
          const float f = a.v_norm ? rn : 1.0f;
          uint16_t* dst = a.v_out + (isk ? t * a.n_k + r - a.n_q : t * a.n_v + r - a.n_q - a.n_k) * D;
          u16x4 oa, ob;
#pragma unroll
          for (int i = 0; i < 4; i++) oa[i] = f32_to_bf16(x[i] * f), ob[i] = f32_to_bf16(x[i + 4] * f);
          *reinterpret_cast<u16x4_a2*>(dst + da) = oa;
          *reinterpret_cast<u16x4_a2*>(dst + db) = ob;
        }
      }
    }
  }
}

template <int D>
hipError_t launch_norm_rope_t(NormRopeArgs& a, int cus, hipStream_t s) {
  constexpr int RPW = 64 / (D / 8), kWaves = kNrThreads / 64;
  const int groups = (a.n_q + a.n_k + a.n_v + RPW - 1) / RPW;
  // a token's rows in as many parts as give every SIMD of the chip two waves
  const int64_t want = (int64_t)cus * 8;
  int64_t chunks = (want + a.n_tokens - 1) / a.n_tokens;
  a.chunks = (int32_t)(chunks > groups ? groups : chunks);
  const int64_t wgs = (a.n_tokens * a.chunks + kWaves - 1) / kWaves;
  // Work-groups that are resident at once (98 registers: five waves a SIMD);
  // they take the tasks in turn, so that the frequencies are computed once each.
  const int64_t most = (int64_t)cus * 5;
  hipLaunchKernelGGL((norm_rope_kernel<D>), dim3((unsigned)(wgs < most ? wgs : most)), dim3(kNrThreads), 0,
                     s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_norm_rope(NormRopeArgs& a, int head_dim, int cus, hipStream_t s) {
  if (head_dim == 128) return launch_norm_rope_t<128>(a, cus, s);
  if (head_dim == 256) return launch_norm_rope_t<256>(a, cus, s);
  if (head_dim == 512) return launch_norm_rope_t<512>(a, cus, s);
  return hipErrorInvalidValue;
}

}  // namespace fmkv
