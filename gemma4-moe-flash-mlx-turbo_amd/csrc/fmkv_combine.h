// The merge of a sequence's split partials, for the kernels that end a decode
// attention call.
#pragma once
#include "fmkv_attn_common.h"

namespace fmkv {
namespace {

// out[seq][h][d] = sum_s 2^(m_s - M) O_s[d] / sum_s 2^(m_s - M) l_s.
// One work-group per (64 dims, q head, sequence); thread (sl, dq) owns dims
// d0 + 4*dq .. +3 and splits sl, sl + 16, ..., merged in one pass with a
// running maximum; the 16 partial merges meet in LDS.
// `dims`: which 64 of head_dim. n_cols: split partials per sequence (splits and
// new-token column), or -1 for per-sequence counts from the struct (a paged batch),
// a shared prefix's partials among them (kTiles); flags: bit 0 f32 output, bit 1 sparse-V,
// bits 8-31 q heads.
template <int D>
__device__ inline void combine_rows(const float* part_o, const float* part_ml, void* out,
                                    int32_t n_cols, int32_t part_stride, uint32_t flags,
                                    const AttnArgs& a, int dims, int h, int seq, int n_seqs) {
  __shared__ float4_t red_o[16][16];
  __shared__ float red_m[16][16];
  __shared__ float red_l[16][16];
  const int tid = threadIdx.x;
  const int dq = tid & 15, sl = tid >> 4;
  const int d0 = dims * 64 + dq * 4;
  const int nqh = (int)(flags >> 8);
  int n_splits = n_cols, s0 = 0;
  if (n_cols < 0) {
    const int64_t T = a.seq_lens ? (int64_t)a.seq_lens[seq] : a.seq_len;
    const SeqGeom geo =
        a.win > 0 ? attn_window(a, seq, T).geo
                  : seq_geometry(T, a.window, a.vis_begin, a.st.table_stride, a.st.block_table != nullptr);
    n_splits = n_splits_for(geo, a.bps0, a.bps, a.max_splits, a.skew_p) + a.new_col;
    if (a.prefix.lens) {
      n_splits += a.prefix.slots;
      if (a.prefix.end(seq, T - a.new_col, a.st.table_stride) == 0) s0 = a.prefix.slots;
    }
  }
  const int64_t stride = (int64_t)nqh;
  const int64_t base = (int64_t)seq * part_stride * stride + h;

  // split maxima are finite (the split kernel starts from -1e30): the first
  // merge scales the empty state by exp2(-inf) = 0
  float M = -INFINITY, den = 0.0f;
  float4_t acc = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = s0 + sl; s < n_splits; s += 16) {
    const int64_t r = base + s * stride;
    const float2 ml = *reinterpret_cast<const float2*>(part_ml + r * 2);
    const float4_t ov = *reinterpret_cast<const float4_t*>(part_o + r * D + d0);
    const float mn = fmaxf(M, ml.x);
    const float alpha = exp2f(M - mn);
    const float w = exp2f(ml.x - mn);
    den = fmaf(w, ml.y, den * alpha);
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = fmaf(w, ov[i], acc[i] * alpha);
    M = mn;
  }
  red_o[sl][dq] = acc;
  red_m[sl][dq] = M;
  red_l[sl][dq] = den;
  __syncthreads();
  if (tid < 16) {
    float Mx = red_m[0][tid];
#pragma unroll
    for (int k = 1; k < 16; k++) Mx = fmaxf(Mx, red_m[k][tid]);
    float4_t s = (float4_t){0.f, 0.f, 0.f, 0.f};
    float L = 0.0f;
    if (Mx != -INFINITY) {
#pragma unroll
      for (int k = 0; k < 16; k++) {
        const float w = exp2f(red_m[k][tid] - Mx);  // 0 for slots without splits (-inf)
        s += w * red_o[k][tid];
        L = fmaf(w, red_l[k][tid], L);
      }
    }
    const int64_t o_idx = ((int64_t)seq * nqh + h) * D + dims * 64 + tid * 4;
    // sparse-V: the kept weights are normalised by the full sum L of the
    // stats pass (no renormalisation, gemma4_attention.rs:226-232), taken at
    // its max M
    const bool sparse = (flags & 2u) != 0;
    float gated = 0.0f;
    if (sparse) {
      const int64_t nh = (int64_t)n_seqs * nqh, r = (int64_t)seq * nqh + h;
      const float Mf = a.tau_stats[nh + r], Lf = a.tau_stats[2 * nh + r];
      gated = (Lf > 0.0f && Mx != -INFINITY) ? exp2f(Mx - Mf) / Lf : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float v = sparse ? s[i] * gated : (L > 0.0f ? s[i] / L : 0.0f);
      if (flags & 1u)
        reinterpret_cast<float*>(out)[o_idx + i] = v;
      else
        reinterpret_cast<uint16_t*>(out)[o_idx + i] = f32_to_bf16(v);
    }
  }
}

}  // namespace
}  // namespace fmkv
