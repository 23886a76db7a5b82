// Pages of a pool moved and compacted.
//
// copy_blocks_kernel: whole blocks (all KV heads) to other blocks of the same
// pool, the same list for the pools of several layers in one launch. A copy is
// bound by memory: each byte read once and written once.
//
// compact_kernel: the tokens that a sequence keeps move to the front of other
// pages. Tokens share cache lines with their neighbours (K codes lie in pieces
// of 16 bytes, V codes of four tokens in one word), so a block some of whose
// tokens are kept is read whole or nearly so; bound by that and the writes.
#include <type_traits>

#include "fmkv_device.h"
#include "fmkv_internal.h"

namespace fmkv {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) Word2 {  // a word at a multiple of 2 bytes
  uint32_t w;
};

constexpr int kCompactThreads = 256;
// A thread copies one piece of 16 bytes: short work-groups start at once on a
// small call, and the chip holds enough of them for a large one. Both accesses
// bypass the caches' reuse order (nontemporal), since neither side is read again
// soon. 5 pools x 1501 pairs of 36.8 KB (553 MB moved): 102.0 us, 5.4 TB/s, what
// a copy of one large buffer reaches; with 2 pieces 104.5, with 4 105.5, with
// temporal accesses 110.6; 9 pairs of 34.8 KB: 2.3 us in a graph, with 4 pieces 2.8.
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = kCopyThreads * 16;

// grid (4 KiB of a block within a pair, pool): a.parts work-groups per pair
__global__ __launch_bounds__(kCopyThreads) void copy_blocks_kernel(CopyArgs a) {
  const int pool = blockIdx.y;
  const uint32_t pair = blockIdx.x / (uint32_t)a.parts, part = blockIdx.x - pair * (uint32_t)a.parts;
  const int32_t src = a.src[pair], dst = a.dst[pair];
  const int32_t n = a.n_blocks[pool];
  if (src < 0 || src >= n || dst < 0 || dst >= n || src == dst) return;
  const int64_t size = a.block_bytes[pool];
  const uint8_t* s = a.base[pool] + src * size;
  uint8_t* d = a.base[pool] + dst * size;
  const int64_t off = (int64_t)part * kCopyBytes + threadIdx.x * 16;
  if (off >= size) return;
  __builtin_nontemporal_store(__builtin_nontemporal_load(reinterpret_cast<const u32x4*>(s + off)),
                              reinterpret_cast<u32x4*>(d + off));
}

template <class T>
__device__ inline T load_at(const uint8_t* block, int64_t at) {
  return *reinterpret_cast<const T*>(block + at);
}

// One work-group per (block of the compacted sequence, KV head, sequence). Its
// 16 tokens' sources are found first (kept position, page); then the block's
// items are gathered, nearly every wave's of one kind (K pieces, V pieces, scales or
// norms), so that a small block does not leave waves idle kind by kind:
//   K: a token's piece is a piece of the source token, whole;
//   V: a piece holds several tokens of some dims, merged from their sources'.
// A token that is not there (past the sequence's list, a position or page out of
// range) leaves its slot as it was; its loads read the block written instead,
// so that no load waits for a test of another. Few registers (26 to 57) and no
// loop over blocks: what is in flight comes from the many work-groups of a CU. 8
// sequences of 3000 to 16000 tokens, every second kept, 8 bits, 2 heads of 512
// dims: 52 us for 186 MB read (the sources' lines, nearly all) and 83 written, 5.1
// TB/s; one of 3077 tokens, a third kept, bf16, 4 heads of 128 dims: 3.9 us in a graph.
template <int MODE, int BITS, int D>
__global__ __launch_bounds__(kCompactThreads) void compact_kernel(CompactArgs a) {
  constexpr BlockLayout L = make_layout(D, BITS, MODE);
  const int seq = blockIdx.z, kvh = blockIdx.y, tid = threadIdx.x;
  int n = a.n_keep[seq];
  if (n > a.max_keep) n = a.max_keep;
  const int first = (int)blockIdx.x * kBlockTokens;
  if (first >= n) return;
  const int32_t dphys = a.dst_table[(int64_t)seq * a.dst_stride + blockIdx.x];
  if (dphys < 0 || dphys >= a.st.n_blocks) return;
  uint8_t* const base = a.st.base + (int64_t)kvh * a.st.head_stride;
  const int64_t doff = dphys * a.st.block_stride;
  uint8_t* const dst = base + doff;

  // the tokens' sources: head-block offset and slot (absent: the block written, -1)
  __shared__ int64_t s_off[kBlockTokens];
  __shared__ int s_tok[kBlockTokens];
  if (tid < kBlockTokens) {
    int64_t off = doff;
    int t = -1;
    if (first + tid < n) {
      const int32_t pos = a.keep[(int64_t)seq * a.max_keep + first + tid];
      if (pos >= 0 && pos / kBlockTokens < a.st.table_stride) {
        const int32_t phys = a.st.block_table[(int64_t)seq * a.st.table_stride + pos / kBlockTokens];
        if (phys >= 0 && phys < a.st.n_blocks) {
          off = phys * a.st.block_stride;
          t = pos & (kBlockTokens - 1);
        }
      }
    }
    s_off[tid] = off;
    s_tok[tid] = t;
  }
  __syncthreads();

  // items: K, V, then scales (or norms) of both
  constexpr int kK = MODE == kCodebook ? D * BITS / 4 : D * BITS / 8;  // pieces of 8 or 16 bytes
  constexpr int kV = MODE == kCodebook ? D : MODE == kPlain ? 2 * D : D * BITS / 8;
  constexpr int kM = MODE == kAffine ? 2 * (D / kGroup) * kBlockTokens : MODE == kCodebook ? 2 * kBlockTokens : 0;
#pragma unroll
  for (int it = 0; it < kK + kV + kM; it += kCompactThreads) {
    const int item = it + tid;
    if (item < kK) {
      // the token, and the piece's place but for the token
      constexpr int kPer = MODE == kPlain ? D / 8 : MODE == kCodebook ? D * BITS / 128 : 1;  // pieces in a row
      constexpr int kHalf = kPer * kBlockTokens;  // plain: the region; codebook: a half
      const int t = MODE == kAffine ? item & 15 : item % kHalf / kPer;
      const int ts = s_tok[t];
      const int shift = (ts < 0 ? 0 : ts - t) * kPer;
      typedef uint32_t piece_t __attribute__((ext_vector_type(MODE == kCodebook ? 2 : 4)));
      const piece_t v = load_at<piece_t>(base + s_off[t], L.k_codes + (item + shift) * (int)sizeof(piece_t));
      if (ts >= 0)
        __builtin_nontemporal_store(v, reinterpret_cast<piece_t*>(dst + L.k_codes + item * (int)sizeof(piece_t)));
    } else if (item < kK + kV) {
      const int i = item - kK;
      if constexpr (MODE == kAffine) {  // (chunk, token quad, dim)
        // bits of a quad's first token in each word, and how far token r's lie
        constexpr uint32_t kOne = BITS == 8 ? 0xffu : 0x0f0fu;
        auto at = [](int r) { return BITS == 8 ? 8 * r : (r >> 1) * 4 + (r & 1) * 16; };
        const int q = (i >> 4) & 3;
        u32x4 v[4], o = (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int ts = s_tok[4 * q + r];
          v[r] = load_at<u32x4>(base + s_off[4 * q + r], L.v_codes + ((i & ~63) + (ts < 0 ? q : ts >> 2) * 16 + (i & 15)) * 16);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int ts = s_tok[4 * q + r];
          const int from = ts < 0 ? at(r) : at(ts & 3);
#pragma unroll
          for (int w = 0; w < 4; w++) o[w] |= (v[r][w] >> from & kOne) << at(r);
        }
        __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(dst + L.v_codes + i * 16));
      } else if constexpr (MODE == kPlain) {  // (dim, half of the tokens)
        const int half = i & 1, d = i >> 1;
        u32x4 o;
#pragma unroll
        for (int r = 0; r < 8; r++) {
          const int t = half * 8 + r, ts = s_tok[t];
          const uint32_t x = load_at<uint16_t>(base + s_off[t], L.v_codes + d * 32 + (ts < 0 ? t : ts) * 2);
          o[r >> 1] = r & 1 ? o[r >> 1] | x << 16 : x;
        }
        *reinterpret_cast<u32x4*>(dst + L.v_codes + d * 32 + half * 16) = o;
      } else {  // a dim's 16 indices, 2 * BITS bytes
        uint64_t o = 0;
#pragma unroll
        for (int t = 0; t < kBlockTokens; t++) {
          // the 4 bytes that hold the index, within the dim's own
          const int ts = s_tok[t], bit = (ts < 0 ? t : ts) * BITS;
          int b = bit >> 4 << 1;
          if (b > 2 * BITS - 4) b = 2 * BITS - 4;
          const uint32_t w = load_at<Word2>(base + s_off[t], L.v_codes + i * 2 * BITS + b).w;
          o |= (uint64_t)(w >> (bit - 8 * b) & ((1u << BITS) - 1u)) << t * BITS;
        }
        uint16_t* p = reinterpret_cast<uint16_t*>(dst + L.v_codes + i * 2 * BITS);
#pragma unroll
        for (int w = 0; w < BITS; w++) p[w] = (uint16_t)(o >> 16 * w);
      }
    } else if (item < kK + kV + kM) {
      constexpr int kOf = kM > 1 ? kM / 2 : 1;  // of K, or of V
      const int v = (item - kK - kV) / kOf, i = (item - kK - kV) - v * kOf, t = i & 15, ts = s_tok[t];
      typedef std::conditional_t<MODE == kAffine, uint32_t, uint16_t> meta_t;
      const int64_t at = (v ? L.v_meta : L.k_meta) + i * (int)sizeof(meta_t);
      const meta_t m = load_at<meta_t>(base + s_off[t], at + (ts < 0 ? 0 : ts - t) * (int)sizeof(meta_t));
      if (ts >= 0) *reinterpret_cast<meta_t*>(dst + at) = m;
    }
  }
}

template <int MODE, int BITS>
hipError_t launch_compact_t(const CompactArgs& a, int n_seqs, hipStream_t s) {
  const dim3 grid((a.max_keep + kBlockTokens - 1) / kBlockTokens, a.st.n_kv_heads, n_seqs);
  const int D = a.st.layout.head_dim;
  const auto kernel = D == 128   ? compact_kernel<MODE, BITS, 128>
                      : D == 256 ? compact_kernel<MODE, BITS, 256>
                                 : compact_kernel<MODE, BITS, 512>;
  hipLaunchKernelGGL(kernel, grid, dim3(kCompactThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_copy_blocks(CopyArgs& a, int n_pools, int64_t n_pairs, hipStream_t s) {
  int64_t most = 0;
  for (int i = 0; i < n_pools; i++) most = a.block_bytes[i] > most ? a.block_bytes[i] : most;
  a.parts = (int32_t)((most + kCopyBytes - 1) / kCopyBytes);
  // pairs of a launch: its grid's x holds fewer than 2^32 threads
  const int64_t per = (int64_t)(UINT32_MAX / kCopyThreads) / a.parts;
  for (int64_t done = 0; done < n_pairs; done += per) {
    const int64_t n = n_pairs - done < per ? n_pairs - done : per;
    const dim3 grid((unsigned)(n * a.parts), n_pools);
    hipLaunchKernelGGL(copy_blocks_kernel, grid, dim3(kCopyThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.src += n;
    a.dst += n;
  }
  return hipSuccess;
}

hipError_t launch_compact(const CompactArgs& a, int n_seqs, hipStream_t s) {
  const BlockLayout& L = a.st.layout;
  if (L.mode == kAffine)
    return L.bits == 4 ? launch_compact_t<kAffine, 4>(a, n_seqs, s)
                       : launch_compact_t<kAffine, 8>(a, n_seqs, s);
  if (L.mode == kPlain) return launch_compact_t<kPlain, 16>(a, n_seqs, s);
  return L.bits == 2   ? launch_compact_t<kCodebook, 2>(a, n_seqs, s)
         : L.bits == 3 ? launch_compact_t<kCodebook, 3>(a, n_seqs, s)
                       : launch_compact_t<kCodebook, 4>(a, n_seqs, s);
}

}  // namespace fmkv
