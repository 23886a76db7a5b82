// Accumulated attention weights of a prompt's queries: weight[s][j] of position j
// is the sum, over the queries of sequence s at positions p >= j and over the query
// heads h, of 2^(s_ph(j) - M_ph) / L_ph, where s are the base-2 scores q . k, M_ph and
// L_ph the maximum and the sum of a query's softmax. V is not read.
//
// M and L are known only when a row has seen all its keys, and the scores of all rows
// with all keys are too many to keep (4 bytes for each pair: 268 MB for 128 queries of
// 16 heads over 32768 keys), so the products are formed twice: a launch for each
// range of keys' (m, l), one for the weights with M and 1 / L merged from those, and
// one that adds up what KV heads and tiles of rows have given a position.
//
// A work-group holds 64 rows (64 / G consecutive queries of a KV head's G heads) as
// matrix-core operands in LDS, rotated in a launch of their own where they are many (four
// prompts of 700 .. 8000 positions, 33 queries, 8 bits, 2 heads of 512 dims: 99.8 us a call with the
// rotation in each work-group, 78.4 without); its waves take different keys, NB blocks of 16 a step,
// straight from memory to registers, where a code is turned into an operand once
// for all rows. Nothing is exchanged between the waves while they run. Over the
// 64-dim groups of a step the scores of the 64 rows with the step's keys stay in
// registers; an operand of the rows is read from LDS once for NB products.
//
// Operands as in prefill (fmkv_prefill.hip): K codes (or centroids) exact, q_rot as
// an f16 high part and residual; plain caches bf16 as stored.
//
// Bound by the issue of matrix and vector instructions, which hardly overlap in two waves a
// SIMD (128 queries of 16 heads over 32768 keys, 4 bits, 8 heads of 256 dims: 79.5 us a launch, 0.86
// PFLOP/s on the matrix cores, busy 48% of the cycles, vector issue 39% and 36%); calls of few steps by their first
// loads and last merges. Priorities of waves, a later start for half of them, and one tile's products
// under the scales of the one before changed nothing.
//
// In the second launch a lane's sums over its rows of the weights of its keys stay in
// registers until all rows are done; 16 lanes meet at the end. Every sum has one
// order: no atomics.
#include <algorithm>
#include <type_traits>

#include "fmkv_device.h"
#include "fmkv_internal.h"
#include "fmkv_rows_common.h"
#include "fmkv_cb_common.h"

namespace fmkv {
namespace {

constexpr int kObRows = 64;
constexpr float kObSlack = 8.0f;  // (base 2) a score may exceed its row's reference by

// Affine caches hold q_rot (times kCodeScale), its sums over 64 dims and those times the codes'
// offset as f16 operands. A row in which one of them would come near f16's largest value, 65504
// (|q_rot|, or a sixteenth of a sum's offset part, past 4000), is held as so much less by a power
// of 2, and its scores are multiplied back in f32: a row of any size has finite operands.
constexpr float kObMost = 4000.0f;

// Blocks of a wave's step in calls of many keys: what the registers hold.
constexpr int many_blocks(int mode) { return mode == kAffine ? 3 : 4; }

template <int D, int BITS, int MODE, int RT>
struct ObPlan {
  static constexpr BlockLayout L = make_layout(D, BITS, MODE);
  static constexpr int NG = D / 64, E = D / 64;
  static constexpr int NW = 8;  // waves: two a SIMD, what their registers allow
  static constexpr int kParts = MODE == kPlain ? 1 : 2;  // high parts, residuals
  // An operand's place: part, tile of rows, 32 dims. 16 bytes more than its 1 KiB: the
  // lanes that write a row, whose pieces lie in as many operands, then take all banks
  // and not the same few (512 dims, a
  // work-group's 64 rows and one step of keys: 28.0 -> 26.3 us).
  static constexpr int kOperands = kParts * RT * 2 * NG;
  static constexpr int kStride = 1040;
  static constexpr int index(int part, int rt, int e) { return (part * RT + rt) * 2 * NG + e; }
  static constexpr int operand(int part, int rt, int e) { return index(part, rt, e) * kStride; }
  static constexpr int kSums = kOperands * kStride;  // the operands of the biases
  static constexpr int kRows = kSums + (MODE == kAffine ? RT * 1024 : 0);
  static constexpr int KW = MODE == kAffine ? BITS / 2 : MODE == kPlain ? 8 : BITS == 3 ? 4 : 2;
  static constexpr int kLut = MODE == kCodebook ? CbLut<BITS == 16 ? 2 : BITS>::kBytes : 16;
  // A tile's operands in memory, as a launch of their own leaves them: 1 KiB each, the biases' last.
  static constexpr int kPieces = kOperands + (MODE == kAffine ? RT : 0);
  // The powers of 2 of the rows behind them.
  static constexpr int kTile = kPieces * 1024 + (MODE == kAffine ? kObRows * 4 : 0);
};

// Calls of more than 16 rows rotate them in a launch of their own, which every range
// of keys of both launches then copies to LDS; where 16 rows are all, or none is rotated
// (plain caches), each work-group prepares them itself.
template <int MODE, int RT>
constexpr bool kObRotated = MODE != kPlain && RT > 1;

// Sequence s of a call: its positions, its keys' blocks, and the WG-steps (NW waves'
// NB blocks) of a range.
struct ObSeq {
  int64_t p0, T;
  int blocks, per;
};
template <int NW, int NB>
__device__ inline ObSeq ob_seq(const ObserveArgs& a, int seq) {
  ObSeq r;
  r.p0 = ((cint_ptr)(uintptr_t)a.start_pos)[seq];
  r.T = r.p0 + a.n_q;
  int64_t b = r.T > 0 ? (r.T + kBlockTokens - 1) / kBlockTokens : 0;
  if (b > a.blocks) b = a.blocks;
  r.blocks = (int)b;
  const int steps = (r.blocks + NW * NB - 1) / (NW * NB);
  r.per = (steps + a.ranges - 1) / a.ranges;
  return r;
}

// Row r of a tile, rotated but for the signs (x: the lane's D / 64 dims), as its places
// in the operands: at `ops`, OP bytes apart, and `sums`. ups: the rows' powers of 2 (affine).
template <int D, int BITS, int MODE, int RT, int OP>
__device__ inline void store_row(const float (&x)[D / 64], uint8_t* ops, uint8_t* sums, float* ups, int r,
                                 int lane, uint32_t sbits, float cs_lane) {
  using P = ObPlan<D, BITS, MODE, RT>;
  constexpr int E = P::E, LPG = 64 / E;  // lanes of a 64-dim group
  const int rt = r >> 4, rc = r & 15, d0 = lane * E, o = d0 & 63;
  float gs = 0.0f, v[E];
  _Float16 hv[E], lv[E];
#pragma unroll
  for (int i = 0; i < E; i++) {
    v[i] = apply_sign(x[i] * cs_lane, sbits, i);
    gs += v[i];
  }
  if constexpr (MODE == kAffine) {
    gs = group_sum<LPG>(gs, lane);
    float most = fabsf(gs) * (kCodeOffset<BITS> / 16.0f), up = 1.0f;
#pragma unroll
    for (int i = 0; i < E; i++) most = fmaxf(most, fabsf(v[i]));
    if (__any(most > kObMost)) {
      most = group_max<64>(most, lane);
      if (most < INFINITY) {  // to [2^10, 2^11)
        const uint32_t e = (__float_as_uint(most) >> 23) - 127u - 10u;
        const float down = __uint_as_float((127u - e) << 23);
        up = __uint_as_float((127u + e) << 23);
        gs *= down;
#pragma unroll
        for (int i = 0; i < E; i++) v[i] *= down;
      }
    }
    if (lane == 0) ups[r] = up;
  }
#pragma unroll
  for (int i = 0; i < E; i++) {
    hv[i] = (_Float16)v[i];
    lv[i] = (_Float16)(v[i] - (float)hv[i]);
    if constexpr (MODE == kAffine) {  // (exact)
      hv[i] = hv[i] * (_Float16)kCodeScale<BITS>;
      lv[i] = lv[i] * (_Float16)kCodeScale<BITS>;
    }
  }
  // (K's operand places: QSlot for affine caches, dims in order for codebooks)
  const int g = d0 >> 6;
  const int s = MODE == kAffine && BITS == 8 ? (o >> 3) & 1 : o >> 5;
  const int jj = MODE == kAffine && BITS == 8 ? o >> 4 : (o >> 3) & 3;
  uint8_t* p = ops + (jj * 16 + rc) * 16 + (o & 7) * 2;
  store_halves<E>(p + P::index(0, rt, 2 * g + s) * OP, hv);
  store_halves<E>(p + P::index(1, rt, 2 * g + s) * OP, lv);
  if constexpr (MODE == kAffine) {
    if ((lane & (LPG - 1)) == 0) {
      // sums of 64 dims, high parts and residuals, against the biases; and
      // the sums that the codes' offset adds, against the scales
      _Float16* q = reinterpret_cast<_Float16*>(sums + rt * 1024) + rc * 8 + g;
      const float off = gs * -kCodeOffset<BITS>;
      const _Float16 h = (_Float16)gs, ho = (_Float16)off;
      q[0] = h;
      q[16 * 8] = (_Float16)(gs - (float)h);
      q[32 * 8] = ho;
      q[48 * 8] = (_Float16)(off - (float)ho);
    }
  }
}

// A tile's rows as operands (kObRotated), 16 rows a work-group, four of its waves' four at a
// time. Grid (tile and 16 rows, KV head, sequence).
template <int D, int BITS, int MODE>
__global__ __launch_bounds__(256) void observe_rows_kernel(ObserveArgs a) {
  constexpr int RT = kObRows / 16;
  using P = ObPlan<D, BITS, MODE, RT>;
  constexpr int E = P::E, NG = P::NG;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x / RT, rt = blockIdx.x % RT, kvh = blockIdx.y, seq = blockIdx.z;
  const int G = a.group, QP = kObRows / G, qi0 = tile * QP;
  const int rows = (a.n_q - qi0 < QP ? a.n_q - qi0 : QP) * G;
  uint8_t* const ops = a.rows + (((int64_t)seq * a.st.n_kv_heads + kvh) * a.tiles + tile) * P::kTile;
  uint8_t* const sums = ops + P::kOperands * 1024;
  float* const ups = reinterpret_cast<float*>(ops + P::kPieces * 1024);
  const uint32_t sbits = lane_sign_bits<D>(a.sign_bits, lane);
  const float cs_lane = fwht_lane_sign(lane) * a.c;
  const int r0 = rt * 16 + wave * 4;
  uint32_t raw[4][E / 2];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int r = r0 + k < rows ? r0 + k : rows - 1, rq = r / G;
    const int64_t row = ((int64_t)seq * a.n_q + qi0 + rq) * a.n_q_heads + (int64_t)kvh * G + (r - rq * G);
    load_words<E / 2>(a.q + row * D + lane * E, raw[k]);
  }
#pragma unroll
  for (int k = 0; k < 4; k++) {
    float x[E];
#pragma unroll
    for (int i = 0; i < E / 2; i++) {
      const uint32_t w = r0 + k < rows ? raw[k][i] : 0u;
      x[2 * i] = __uint_as_float(w << 16) * a.qscale;
      x[2 * i + 1] = __uint_as_float(w & 0xffff0000u) * a.qscale;
    }
    wave_fwht_signed<E>(x, lane);
    store_row<D, BITS, MODE, RT, 1024>(x, ops, sums, ups, r0 + k, lane, sbits, cs_lane);
    if (MODE == kAffine && NG < 8 && lane < 4 * (8 - NG))  // (groups that the dims do not have)
      reinterpret_cast<_Float16*>(sums + rt * 1024)[(lane & 3) * 128 + ((r0 + k) & 15) * 8 + NG + (lane >> 2)] =
          (_Float16)0.0f;
  }
}

// SUMS: the second launch. Grid (range of keys, KV head and sharer of its tiles, sequence).
// RT: matrix-core tiles of the rows, 4, or 1 where all calls' tiles have 16 rows at most.
template <int D, int BITS, int MODE, int RT, int NB, bool SUMS>
__global__ __launch_bounds__((ObPlan<D, BITS, MODE, RT>::NW * 64))
__attribute__((amdgpu_waves_per_eu(2, 2)))
void observe_kernel(ObserveArgs a) {
  using P = ObPlan<D, BITS, MODE, RT>;
  constexpr BlockLayout L = P::L;
  constexpr int NG = P::NG, NW = P::NW, E = P::E, KW = P::KW;
  constexpr int CB = MODE == kCodebook ? BITS : 2;
  __shared__ __align__(16) uint8_t rows_s[P::kRows];
  __shared__ __align__(16) uint8_t lut[P::kLut];
  __shared__ int row_pos[RT * 16];
  __shared__ float row_up[MODE == kAffine ? RT * 16 : 1];
  __shared__ float2 stat[SUMS ? 1 : NW][RT * 16];  // (m, l) of the waves; SUMS: M, 1 / L

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane >> 4, c = lane & 15;
  const int seq = blockIdx.z, range = blockIdx.x;
  const int kvh = blockIdx.y / a.sharers, sharer = blockIdx.y - kvh * a.sharers;
  const ObSeq q = ob_seq<NW, NB>(a, seq);
  const int s_begin = range * q.per;
  const int n_steps = (q.blocks + NW * NB - 1) / (NW * NB);
  const int s_end = s_begin + q.per < n_steps ? s_begin + q.per : n_steps;
  if (s_begin >= s_end) return;
  const int ranges = (n_steps + q.per - 1) / q.per;  // of this sequence
  const int G = a.group, QP = kObRows / G;

  const uint64_t base = reinterpret_cast<uint64_t>(a.st.base) + kvh * a.st.head_stride;
  const cint_ptr table = (cint_ptr)(uintptr_t)(a.st.block_table + (int64_t)seq * a.st.table_stride);
  const int32_t n_pool = (int32_t)(a.st.n_blocks < INT32_MAX ? a.st.n_blocks : INT32_MAX);
  auto blk_ptr = [&](int b) __attribute__((always_inline)) -> gptr_t {
    // (past the last block: that one, whose keys are masked; an entry outside the
    // pool reads a valid block rather than faulting)
    const int32_t e = table[b < q.blocks ? b : q.blocks - 1];
    const uint32_t phys = (uint32_t)(e < 0 ? 0 : (e >= n_pool ? n_pool - 1 : e));
    return (gptr_t)(base + (uint64_t)phys * (uint64_t)a.st.block_stride);
  };

  const int kbit = (c * (D / 2) + 8 * j) * CB;
  const uint32_t ksh = kbit & 31;
  const uint32_t k_off = (uint32_t)L.k_codes + (MODE == kAffine     ? lane * 16
                                                : MODE == kCodebook ? (kbit >> 5) * 4
                                                                    : (c * D + 8 * j) * 2);
  const uint32_t km_off = (uint32_t)L.k_meta + j * 16;
  const uint32_t kb_off = (uint32_t)L.k_meta + c * 4 + (j < 2 ? 2 : 0);
  const U4Consts u4;
  struct Stage {
    uint32_t kr[NB][KW];
    u32x4 km[NB];
  };
  // affine: the biases (lanes (0, c), (1, c)) or scales of key c of each block, by group
  auto load_bias = [&](const gptr_t (&bp)[NB], half8_t (&x)[NB]) __attribute__((always_inline)) {
    if constexpr (MODE == kAffine) {
#pragma unroll
      for (int b = 0; b < NB; b++) {
        x[b] = half8_t{};
#pragma unroll
        for (int g = 0; g < NG; g++) x[b][g] = load_at<_Float16>(bp[b], kb_off, g * 64);
      }
    }
  };
  auto load = [&](const gptr_t (&bp)[NB], int g, Stage& st) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < NB; b++) {
      if constexpr (MODE == kAffine) {
        if constexpr (BITS == 8) {
          const u32x4 w = load_at<u32x4>(bp[b], k_off, g * 1024);
#pragma unroll
          for (int i = 0; i < 4; i++) st.kr[b][i] = w[i];
        } else {
          const u32x2 w = load_at<u32x2>(bp[b], k_off, (g >> 1) * 1024 + (g & 1) * 8);
          st.kr[b][0] = w[0];
          st.kr[b][1] = w[1];
        }
        st.km[b] = load_at<u32x4>(bp[b], km_off, g * 64);
      } else if constexpr (MODE == kCodebook) {
        const int off = (g / (NG / 2)) * (D * CB) + (g % (NG / 2)) * 8 * CB;
#pragma unroll
        for (int s = 0; s < 2; s++) {
          if constexpr (CB == 3) {
            const u32x2 w = load_at<u32x2_a4>(bp[b], k_off, off + s * 4 * CB);
            st.kr[b][2 * s] = w[0];
            st.kr[b][2 * s + 1] = w[1];
          } else {
            st.kr[b][s] = load_at<uint32_t>(bp[b], k_off, off + s * 4 * CB);
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < 2; s++) {
          const u32x4 w = load_at<u32x4>(bp[b], k_off, g * 128 + s * 64);
#pragma unroll
          for (int i = 0; i < 4; i++) st.kr[b][4 * s + i] = w[i];
        }
      }
    }
  };

  const uint32_t sbits = lane_sign_bits<D>(a.sign_bits, lane);
  const float cs_lane = fwht_lane_sign(lane) * a.c;
  const uint32_t lut_l = lds_addr(lut) + (lane & (kLutCopies - 1)) * 4;
  if constexpr (MODE == kCodebook) cb_fill_lut<CB>(lut, tid, NW * 64);
  if constexpr (MODE == kAffine && !kObRotated<MODE, RT>) {  // (what of the biases' operands no group fills is 0)
    for (int i = tid; i < RT * 64; i += NW * 64)
      reinterpret_cast<u32x4*>(rows_s + P::kSums)[i] = (u32x4){0, 0, 0, 0};
    __syncthreads();
  }

  bool first = true;  // of this work-group's tiles
  // (the last tile first: it sees the most keys, so every later one's steps have a
  // partial to add to)
#pragma unroll 1
  for (int tile = a.tiles - 1 - sharer; tile >= 0; tile -= a.sharers) {
    const int qi0 = tile * QP;
    const int nq = a.n_q - qi0 < QP ? a.n_q - qi0 : QP;
    const int rows = nq * G;
    const int64_t p_last = q.p0 + qi0 + nq - 1, p_first = q.p0 + qi0;
    const int64_t ml_row = (((int64_t)seq * a.st.n_kv_heads + kvh) * a.tiles + tile) * kObRows;

    auto blocks_of = [&](int step, gptr_t (&bp)[NB]) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < NB; b++) bp[b] = blk_ptr((step * NW + wave) * NB + b);
    };
    gptr_t bp[NB], bn[NB];
    Stage cur, nxt;
    half8_t bias[NB];
    blocks_of(s_begin, bp);
    load(bp, 0, cur);
    load_bias(bp, bias);

    float up = 1.0f;
    if constexpr (kObRotated<MODE, RT>) {
      const uint8_t* image = a.rows + ml_row / kObRows * P::kTile;
      if (MODE == kAffine && tid < RT * 16) up = reinterpret_cast<const float*>(image + P::kPieces * 1024)[tid];
      const u32x4 rs = buffer_rsrc(image, P::kPieces * 1024);
      const uint32_t to = lds_addr(rows_s);
#pragma unroll 1
      for (int o = wave; o < P::kPieces; o += NW)
        dma16(to + (o < P::kOperands ? o * P::kStride : P::kSums + (o - P::kOperands) * 1024),
              o * 1024 + lane * 16, rs);
    }

    // ---- the rows as operands: row r by wave r % NW ----
    for (int r = tid; r < RT * 16; r += NW * 64) {
      const int rq = r / G;
      // (a row past the chunk, or a padded one before position 0, sees nothing)
      const int64_t p = r < rows ? q.p0 + qi0 + rq : -1;
      row_pos[r] = (int)(p < 0 ? -1 : p);
    }
    if constexpr (SUMS) {  // sixteen lanes a row: each merges every sixteenth range, then they meet
      for (int r = tid >> 4; r < RT * 16; r += NW * 4) {
        const float2* x = reinterpret_cast<const float2*>(a.ml) + (ml_row + r) * a.ranges;
        float M = -1e30f, l = 0.0f;
        for (int k = tid & 15; k < ranges; k += 16) {
          const float mn = fmaxf(M, x[k].x);
          l = fmaf(l, exp2f(M - mn), x[k].y * exp2f(x[k].x - mn));
          M = mn;
        }
        const float Mx = group_max<16>(M, lane);
        l = group_sum<16>(l * exp2f(M - Mx), lane);
        if ((tid & 15) == 0) stat[0][r] = make_float2(Mx, l > 0.0f ? 1.0f / l : 0.0f);
      }
    }
    if constexpr (kObRotated<MODE, RT>) {
      if (MODE == kAffine && tid < RT * 16) row_up[tid] = up;
      wait_vmcnt<0>();
    } else {
      // Four rows of a wave at a time, the next four on their way meanwhile
      uint32_t raw[4][E / 2], ahead[4][E / 2];
      auto load_rows = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int rr = r0 + k * NW, r = rr < rows ? rr : rows - 1, rq = r / G;
          const int64_t row = ((int64_t)seq * a.n_q + qi0 + rq) * a.n_q_heads + (int64_t)kvh * G + (r - rq * G);
          load_words<E / 2>(a.q + row * D + lane * E, ahead[k]);
        }
      };
      load_rows(wave);
#pragma unroll 1
      for (int r0 = wave; r0 < RT * 16; r0 += 4 * NW) {
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
          for (int i = 0; i < E / 2; i++) raw[k][i] = r0 + k * NW < rows ? ahead[k][i] : 0u;
        if (r0 + 4 * NW < RT * 16) load_rows(r0 + 4 * NW);
        const int d0 = lane * E, o = d0 & 63;
        float x[4][E];
        if constexpr (MODE != kPlain) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
              x[k][2 * i] = __uint_as_float(raw[k][i] << 16) * a.qscale;
              x[k][2 * i + 1] = __uint_as_float(raw[k][i] & 0xffff0000u) * a.qscale;
            }
            wave_fwht_signed<E>(x[k], lane);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int r = r0 + k * NW, rt = r >> 4, rc = r & 15;
          if (r >= RT * 16) continue;
          if constexpr (MODE == kPlain) {
            const int e = d0 >> 5;
            uint8_t* p = rows_s + P::operand(0, rt, e) + (((o & 31) >> 3) * 16 + rc) * 16 + (o & 7) * 2;
#pragma unroll
            for (int i = 0; i < E / 2; i++) reinterpret_cast<uint32_t*>(p)[i] = raw[k][i];
          } else {
            store_row<D, BITS, MODE, RT, P::kStride>(x[k], rows_s, rows_s + P::kSums, row_up, r, lane, sbits,
                                                        cs_lane);
          }
        }
      }
    }
    __syncthreads();
    // (kObMost; any row of the tile)
    const bool scaled = MODE == kAffine && __any(row_up[lane & (RT * 16 - 1)] != 1.0f);

    int p_row[RT];
    float m_run[RT], l_run[RT];  // SUMS: M and 1 / L of the lane's rows
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      p_row[rt] = row_pos[rt * 16 + c];
      m_run[rt] = -1e30f;
      l_run[rt] = 0.0f;
      if constexpr (SUMS) {
        const float2 x = stat[0][rt * 16 + c];
        m_run[rt] = x.x;
        l_run[rt] = x.y;
        if (scaled) m_run[rt] /= row_up[rt * 16 + c];
      }
    }

    // ---- the steps: NB blocks of keys a wave ----
    // the next products' operands, rows of a tile and 64 dims: residuals, high parts
    half8_t rows_l[2], rows_h[2];
    auto load_tile = [&](half8_t (&x)[2], int part, int rt, int g) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; t++)
        x[t] = *reinterpret_cast<const half8_t*>(
            rows_s + P::operand(part, rt, 2 * g + t) + lane * 16);
    };
    if constexpr (MODE != kPlain) load_tile(rows_l, 1, 0, 0);
    load_tile(rows_h, 0, 0, 0);
#pragma unroll 1
    for (int step = s_begin; step < s_end; step++) {
      const int64_t key0 = (int64_t)(step * NW + wave) * NB * kBlockTokens;
      float* part = nullptr;
      if constexpr (SUMS)
        part = a.part + ((int64_t)seq * a.st.n_kv_heads * a.sharers + blockIdx.y) * a.part_width + key0;
      if (key0 > p_last) {  // nothing of this tile sees these keys, or later ones
        if constexpr (SUMS) {
          if (first)
            for (int i = lane; i < NB * kBlockTokens && key0 + i < a.part_width; i += 64) part[i] = 0.0f;
        }
        continue;
      }
      blocks_of(step + 1 < s_end ? step + 1 : step, bn);
      u32x2 kn[MODE == kCodebook ? NB : 1];
      if constexpr (MODE == kCodebook) {
#pragma unroll
        for (int b = 0; b < NB; b++) kn[b] = load_at<u32x2>(bp[b], (uint32_t)L.k_meta + 8 * j);
      }
      // The scores start at -M (SUMS, affine), and at the biases' and the codes' offset's part, one
      // product of 16 keys' biases and scales (lanes (0, c) and (1, c): key c's biases of groups
      // 0 .. 7, the others its scales) with the rows' sums
      float4_t s[RT][NB];
#pragma unroll
      for (int b = 0; b < NB; b++) {
        half8_t kb{};
        if constexpr (MODE == kAffine) {
#pragma unroll
          for (int g = 0; g < 8; g++) kb[g] = bias[b][g];
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
          const float z = SUMS && MODE == kAffine ? -m_run[rt] : 0.0f;
          s[rt][b] = (float4_t){z, z, z, z};
          if constexpr (MODE == kAffine) {
            const half8_t qb = *reinterpret_cast<const half8_t*>(rows_s + P::kSums + rt * 1024 + lane * 16);
            s[rt][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qb, s[rt][b], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
#pragma unroll
      for (int g = 0; g < NG; g++) {
        if (g + 1 < NG)
          load(bp, g + 1, nxt);
        else
          load(bn, 0, nxt);
        half8_t ah[NB][2], al[NB][2];  // (al: 4-bit codebooks)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int t = 0; t < 2; t++) {
            if constexpr (MODE == kAffine) {
              if constexpr (BITS == 8) {
                const uint32_t w0 = cur.kr[b][2 * t], w1 = cur.kr[b][2 * t + 1];
                ah[b][t] = cat8(u8x2_to_h2_biased(w0, 0x04010400u), u8x2_to_h2_biased(w0, 0x04030402u),
                                u8x2_to_h2_biased(w1, 0x04010400u), u8x2_to_h2_biased(w1, 0x04030402u));
              } else {
                const uint32_t x = cur.kr[b][t];
                ah[b][t] = cat8(u4x2_to_h2_unit(x, 0, u4), u4x2_to_h2_unit(x, 1, u4),
                                u4x2_to_h2_unit(x, 2, u4), u4x2_to_h2_unit(x, 3, u4));
              }
            } else if constexpr (MODE == kPlain) {
              ah[b][t] = __builtin_bit_cast(half8_t, (u32x4){cur.kr[b][4 * t], cur.kr[b][4 * t + 1],
                                                             cur.kr[b][4 * t + 2], cur.kr[b][4 * t + 3]});
            } else {
              uint32_t f;
              if constexpr (CB == 3)
                f = __builtin_amdgcn_alignbit(cur.kr[b][2 * t + 1], cur.kr[b][2 * t], ksh);
              else
                f = cur.kr[b][t] >> ksh;
              if constexpr (kCbExact<CB>) {
                ah[b][t] = __builtin_bit_cast(
                    half8_t, (u32x4){cb_pair_exact<CB, 0>(lut_l, f), cb_pair_exact<CB, 1>(lut_l, f),
                                     cb_pair_exact<CB, 2>(lut_l, f), cb_pair_exact<CB, 3>(lut_l, f)});
              } else {
                uint32_t h4[4], l4[4];
                cb_pair_hl4<0>(lut_l, f, h4[0], l4[0]);
                cb_pair_hl4<1>(lut_l, f, h4[1], l4[1]);
                cb_pair_hl4<2>(lut_l, f, h4[2], l4[2]);
                cb_pair_hl4<3>(lut_l, f, h4[3], l4[3]);
                ah[b][t] = __builtin_bit_cast(half8_t, (u32x4){h4[0], h4[1], h4[2], h4[3]});
                al[b][t] = __builtin_bit_cast(half8_t, (u32x4){l4[0], l4[1], l4[2], l4[3]});
              }
            }
          }
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
          float4_t acc[NB];
#pragma unroll
          for (int b = 0; b < NB; b++) acc[b] = MODE == kAffine ? (float4_t){0.f, 0.f, 0.f, 0.f} : s[rt][b];
          // The residuals' products first; a part's operands of the next tile come as soon
          // as this one's products are under way. (The barriers keep the compiler from
          // starting all tiles of a step at once, which no registers hold.)
          const int rn = rt + 1 < RT ? rt + 1 : 0, gn = rn ? g : g + 1 < NG ? g + 1 : 0;
          auto products = [&](const half8_t (&k)[NB][2], const half8_t (&x)[2]) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
              for (int b = 0; b < NB; b++) {
                if constexpr (MODE == kPlain)
                  acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                      __builtin_bit_cast(bf16x8_t, k[b][t]), __builtin_bit_cast(bf16x8_t, x[t]), acc[b], 0, 0, 0);
                else
                  acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[b][t], x[t], acc[b], 0, 0, 0);
              }
          };
          if constexpr (MODE != kPlain) {
            products(ah, rows_l);
            load_tile(rows_l, 1, rn, gn);
          }
          if constexpr (MODE == kCodebook && !kCbExact<CB>) products(al, rows_h);
          products(ah, rows_h);
          load_tile(rows_h, 0, rn, gn);
          if constexpr (MODE == kAffine) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
              for (int i = 0; i < 4; i++) s[rt][b][i] = fmaf(lo16(cur.km[b][i]), acc[b][i], s[rt][b][i]);
            // (here, not sunk to the softmax with every group's products kept for it)
#pragma unroll
            for (int b = 0; b < NB; b++) asm volatile("" : "+v"(s[rt][b]));
          } else {
#pragma unroll
            for (int b = 0; b < NB; b++) s[rt][b] = acc[b];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        cur = nxt;
      }
#pragma unroll
      for (int b = 0; b < NB; b++) bp[b] = bn[b];
      load_bias(bp, bias);

      if (MODE == kAffine && scaled) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
          for (int b = 0; b < NB; b++) s[rt][b] *= row_up[rt * 16 + c];
      }

      // ---- softmax: lane (j, c) has keys 16 b + 4 j + i of rows 16 rt + c ----
      const bool full = key0 + NB * kBlockTokens - 1 <= p_first && rows == RT * 16 && p_first >= 0;
      float4_t w[SUMS ? NB : 1];
      if constexpr (SUMS) {
#pragma unroll
        for (int b = 0; b < NB; b++) w[b] = (float4_t){0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if constexpr (MODE == kCodebook) {
              const uint32_t n = kn[b][i >> 1];
              s[rt][b][i] *= (i & 1 ? hi16(n) : lo16(n)) * (a.c * kCbOperandScale<CB>);
            }
            if constexpr (MODE == kPlain) s[rt][b][i] *= a.qscale;
          }
        if (!full) {
          const int rel = p_row[rt] - (int)key0 - 4 * j;  // (key0 <= p_last: both fit)
#pragma unroll
          for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (16 * b + i > rel) s[rt][b][i] = -INFINITY;
        }
        if constexpr (SUMS) {
#pragma unroll
          for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              w[b][i] = fmaf(__builtin_amdgcn_exp2f(MODE == kAffine ? s[rt][b][i] : s[rt][b][i] - m_run[rt]),
                             l_run[rt], w[b][i]);
        } else {
          float mx = -INFINITY;
#pragma unroll
          for (int b = 0; b < NB; b++)
            mx = fmaxf(mx, fmaxf(fmaxf(s[rt][b][0], s[rt][b][1]), fmaxf(s[rt][b][2], s[rt][b][3])));
          if (__any(mx > m_run[rt] + kObSlack)) {
            const float m_new = fmaxf(m_run[rt], mx);
            l_run[rt] *= __builtin_amdgcn_exp2f(m_run[rt] - m_new);
            m_run[rt] = m_new;
          }
#pragma unroll
          for (int b = 0; b < NB; b++) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = __builtin_amdgcn_exp2f(s[rt][b][i] - m_run[rt]);
            l_run[rt] += (p[0] + p[1]) + (p[2] + p[3]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);  // (nor all tiles' weights at once)
      }
      if constexpr (SUMS) {  // the sixteen lanes of a key meet; lane c < NB stores block c's
        float4_t mine = w[0];
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
          for (int i = 0; i < 4; i++) w[b][i] = group_sum<16>(w[b][i], lane);
          if (c == b) mine = w[b];
        }
        const int64_t at = 16 * c + 4 * j;
        if (c < NB && key0 + at < a.part_width) {
          float4_t* p = reinterpret_cast<float4_t*>(part + at);
          *p = first ? mine : *p + mine;
        }
      }
    }
    first = false;
    if constexpr (!SUMS) {
      // (m, l) of the lanes' key quarters, then of the waves
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        const float M = xor32_max(xor16_max(m_run[rt]));
        const float l = xor32_sum(xor16_sum(l_run[rt] * __builtin_amdgcn_exp2f(m_run[rt] - M)));
        if (j == 0) stat[wave][rt * 16 + c] = make_float2(M, l);
      }
      __syncthreads();
      if (tid < RT * 16) {
        float M = stat[0][tid].x, l = 0.0f;
#pragma unroll
        for (int w = 1; w < NW; w++) M = fmaxf(M, stat[w][tid].x);
#pragma unroll
        for (int w = 0; w < NW; w++) l = fmaf(stat[w][tid].y, exp2f(stat[w][tid].x - M), l);
        reinterpret_cast<float2*>(a.ml)[(ml_row + tid) * a.ranges + range] = make_float2(M, l);
      }
    }
    __syncthreads();  // the rows and their statistics are done with
  }
}

// weights_out[s][j] = weights_in[s][j] + the partials of position j, in order.
__global__ __launch_bounds__(256) void observe_sum_kernel(ObserveArgs a) {
  const int seq = blockIdx.y;
  int64_t T = (int64_t)a.start_pos[seq] + a.n_q;
  if (T > a.weights_width) T = a.weights_width;
  const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p >= T) return;
  const int n = a.st.n_kv_heads * a.sharers;
  float sum = 0.0f;
  if (p < (int64_t)a.blocks * kBlockTokens) {
    const float* src = a.part + (int64_t)seq * n * a.part_width + p;
#pragma unroll 8
    for (int i = 0; i < n; i++) sum += src[(int64_t)i * a.part_width];
  }
  const int64_t at = (int64_t)seq * a.weights_width + p;
  a.weights_out[at] = (a.weights_in ? a.weights_in[at] : 0.0f) + sum;
}

hipError_t launch_sum(const ObserveArgs& a, hipStream_t s) {
  const int64_t keys = (int64_t)a.blocks * kBlockTokens;
  hipLaunchKernelGGL(observe_sum_kernel, dim3((unsigned)((keys + 255) / 256), a.n_seqs), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int D, int BITS, int MODE, int RT, int NB>
hipError_t launch_ob(const ObserveArgs& a, hipStream_t s) {
  const dim3 grid(a.ranges, a.st.n_kv_heads * a.sharers, a.n_seqs), block(ObPlan<D, BITS, MODE, RT>::NW * 64);
  hipError_t e = hipSuccess;
  if constexpr (kObRotated<MODE, RT>) {
    hipLaunchKernelGGL((observe_rows_kernel<D, BITS, MODE>),
                       dim3(a.tiles * RT, a.st.n_kv_heads, a.n_seqs), dim3(256), 0, s, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  hipLaunchKernelGGL((observe_kernel<D, BITS, MODE, RT, NB, false>), grid, block, 0, s, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((observe_kernel<D, BITS, MODE, RT, NB, true>), grid, block, 0, s, a);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  return launch_sum(a, s);
}
template <int D, int BITS, int MODE>
hipError_t launch_ob(const ObserveArgs& a, hipStream_t s) {
  constexpr int kMany = many_blocks(MODE);
  if (a.n_q * a.group <= 16)
    return a.step_blocks > 1 ? launch_ob<D, BITS, MODE, 1, kMany>(a, s) : launch_ob<D, BITS, MODE, 1, 1>(a, s);
  return a.step_blocks > 1 ? launch_ob<D, BITS, MODE, 4, kMany>(a, s) : launch_ob<D, BITS, MODE, 4, 1>(a, s);
}

}  // namespace

size_t observe_plan(ObserveArgs& a, int cus) {
  constexpr int waves = 8;
  const int64_t places = cus;  // work-groups that run at once
  const int qp = kObRows / a.group;
  a.tiles = (a.n_q + qp - 1) / qp;
  const int64_t per_tile = (int64_t)a.st.n_kv_heads * a.n_seqs;
  const int64_t rows = per_tile * a.tiles;
  const int many = many_blocks(a.st.layout.mode);
  a.step_blocks = rows * ((a.blocks + many * waves - 1) / (many * waves)) >= places ? many : 1;
  const int64_t steps = (a.blocks + waves * a.step_blocks - 1) / (waves * a.step_blocks);
  // as many work-groups as run at once, several tiles one after the other where there are more
  a.sharers = (int32_t)std::clamp<int64_t>(2 * places / per_tile, 1, a.tiles);
  // More ranges than places where sequences are likely ragged: eight of 600 .. 6000
  // positions, 4 bits, 8 heads of 256 dims, 32 queries: 62.7 us with as many, 53.7 with three
  // times as many (two of 3000 .. 9000: 30.0 and 36.9; four of 12000 each, 512 dims: 140 and 160).
  const int ragged = a.n_seqs > 2 ? 3 : 1;
  a.ranges = (int32_t)std::clamp<int64_t>(ragged * places / (per_tile * a.sharers), 1, steps);
  a.part_width = (int64_t)a.blocks * kBlockTokens;
  // operands of a tile: high parts and residuals of 64 rows, 4 KiB for the biases and the powers of 2
  a.images = a.st.layout.mode == kPlain || a.n_q * a.group <= 16
                 ? 0
                 : rows * (kObRows * a.st.layout.head_dim + (a.st.layout.mode == kAffine ? 1024 + kObRows : 0));
  return (size_t)(a.images + rows * a.ranges * kObRows * 2 + per_tile * a.sharers * a.part_width);
}

hipError_t launch_observe(const ObserveArgs& a, hipStream_t s) {
  if (a.n_q == 0) return launch_sum(a, s);  // (of no partials: the weights as they were)
  const BlockLayout& L = a.st.layout;
  if (L.mode == kAffine) {
    switch (L.head_dim * 16 + L.bits) {
      case 128 * 16 + 4: return launch_ob<128, 4, kAffine>(a, s);
      case 128 * 16 + 8: return launch_ob<128, 8, kAffine>(a, s);
      case 256 * 16 + 4: return launch_ob<256, 4, kAffine>(a, s);
      case 256 * 16 + 8: return launch_ob<256, 8, kAffine>(a, s);
      case 512 * 16 + 4: return launch_ob<512, 4, kAffine>(a, s);
      case 512 * 16 + 8: return launch_ob<512, 8, kAffine>(a, s);
    }
  } else if (L.mode == kCodebook) {
    switch (L.head_dim * 16 + L.bits) {
      case 128 * 16 + 2: return launch_ob<128, 2, kCodebook>(a, s);
      case 128 * 16 + 3: return launch_ob<128, 3, kCodebook>(a, s);
      case 128 * 16 + 4: return launch_ob<128, 4, kCodebook>(a, s);
      case 256 * 16 + 2: return launch_ob<256, 2, kCodebook>(a, s);
      case 256 * 16 + 3: return launch_ob<256, 3, kCodebook>(a, s);
      case 256 * 16 + 4: return launch_ob<256, 4, kCodebook>(a, s);
      case 512 * 16 + 2: return launch_ob<512, 2, kCodebook>(a, s);
      case 512 * 16 + 3: return launch_ob<512, 3, kCodebook>(a, s);
      case 512 * 16 + 4: return launch_ob<512, 4, kCodebook>(a, s);
    }
  } else if (L.mode == kPlain) {
    switch (L.head_dim) {
      case 128: return launch_ob<128, 16, kPlain>(a, s);
      case 256: return launch_ob<256, 16, kPlain>(a, s);
      case 512: return launch_ob<512, 16, kPlain>(a, s);
    }
  }
  return hipErrorInvalidValue;
}

}  // namespace fmkv
