// What the kernels of many query rows over a cache share (prefill, accumulated
// weights): matrix-core operands of whole codes, loads at a lane's offset from a
// uniform address.
#pragma once
#include "fmkv_attn_common.h"

namespace fmkv {
namespace {

// K operand of MFMA s of group g as the plain codes (exact f16 integers);
// w: the lane's words of the group.
template <int BITS>
__device__ inline half8_t k_operand_plain(const uint32_t* w, int s) {
  if constexpr (BITS == 8) {
    const uint32_t w0 = w[2 * s], w1 = w[2 * s + 1];
    return cat8(u8x2_to_h2(w0, 0x04010400u), u8x2_to_h2(w0, 0x04030402u),
                u8x2_to_h2(w1, 0x04010400u), u8x2_to_h2(w1, 0x04030402u));
  } else {
    return cat8(u4x2_to_h2(w[s], 0), u4x2_to_h2(w[s], 1), u4x2_to_h2(w[s], 2), u4x2_to_h2(w[s], 3));
  }
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
__device__ inline uint32_t pack_bf16x2(float a, float b) {
  return (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
}

// A uniform address in memory and loads at a lane's offset from it. (Global
// address space: a generic pointer's flat loads also count as LDS operations,
// and every wait for LDS data or at a barrier would wait for memory too.)
typedef const uint8_t __attribute__((address_space(1)))* gptr_t;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_a4 __attribute__((aligned(4)));  // two words at a 4-byte boundary
template <class T>
__device__ inline T load_at(gptr_t p, uint32_t off, int imm = 0) {
  return *reinterpret_cast<const T __attribute__((address_space(1)))*>(p + off + imm);
}

// 2 N consecutive bf16 in one load a lane (aligned to one of them only).
template <int N>
__device__ inline void load_words(const uint16_t* src, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    typedef uint32_t word __attribute__((aligned(2)));
    w[0] = *reinterpret_cast<const word*>(src);
  } else {
    typedef uint32_t vec __attribute__((ext_vector_type(N), aligned(2)));
    const vec v = *reinterpret_cast<const vec*>(src);
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = v[i];
  }
}

// LDS of this wave written, every wave of the work-group here. Loads from
// memory stay in flight across it.
__device__ inline void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Scalar loads of what every lane reads alike.
typedef const int32_t __attribute__((address_space(4)))* cint_ptr;

}  // namespace
}  // namespace fmkv
