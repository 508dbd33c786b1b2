// Pieces shared by the kernels around attention (rotary positions, the 4-bit cache): 16-bit conversions, the record
// of the cache, and the host side of a call.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tcgen05_common.cuh"

namespace rsfa {
namespace {

// ------------------------------------------------------------------ 16-bit numbers
template <bool kBf16>
__device__ __forceinline__ float2 to_f32x2(uint32_t v) {
  if constexpr (kBf16) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
}
template <bool kBf16>
__device__ __forceinline__ float to_f32(uint16_t v) {
  if constexpr (kBf16) return __uint_as_float(static_cast<uint32_t>(v) << 16);
  return __half2float(__ushort_as_half(v));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t from_f32x2(float a, float b) {
  if constexpr (kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <bool kBf16>
__device__ __forceinline__ uint16_t from_f32(float a) {
  if constexpr (kBf16) return __bfloat16_as_ushort(__float2bfloat16_rn(a));
  return __half_as_ushort(__float2half_rn(a));
}

// A bad index found on the device: the first one stays in the status word until it is read.
__device__ __forceinline__ void report_bad_index(int* status, int tag) {
  atomicCAS(status, 0, (kStatusBadIndex << 16) | tag);
}

// ------------------------------------------------------------------ the 4-bit record
// One token of one K/V head, 5 D / 4 bytes: D / 2 bytes of K codes, D / 2 of V codes, then for K and for V one
// (scale, minimum) pair of 16-bit numbers per group of 32 dims.  A value is scale * code + minimum.
// The codes lie in the order in which a lane of an mma.sync fragment wants them, in one load each:
//   K: word (w, c) = the eight dims 32 w + 8 c .. + 7 of group w, one nibble each, and the words of one c together
//      (c = lane % 4 picks the dims of an A fragment whose rows are tokens);
//   V: half word (g, w) = the four dims 32 w + 4 g .. + 3, the half words of one g together
//      (g = lane / 4 picks the rows of an A fragment whose rows are dims).
template <int D>
struct Record {
  static constexpr int kGroups = D / 32;
  static constexpr int kBytes = D * 5 / 4;
  static constexpr int kVCodes = D / 2;
  static constexpr int kKPairs = D;
  static constexpr int kVPairs = D + 4 * kGroups;
  static constexpr int kWordsPerC = kGroups < 4 ? kGroups : 4;   // K words of one c that lie together
  __host__ __device__ static constexpr int k_word(int w, int c) {
    return (w / 4) * 64 + c * 4 * kWordsPerC + 4 * (w % 4);
  }
  __host__ __device__ static constexpr int v_half(int w, int g) { return kVCodes + g * (D / 16) + 2 * w; }
};

// Where slot `slot` of sequence b is: its page and the row in it.  False (and the status word set) for a page
// that the cache does not have.
__device__ __forceinline__ bool find_page(const Cache4& c, int b, int slot, int64_t* page) {
  const int id = c.table[static_cast<int64_t>(b) * c.table_stride + (slot >> c.page_shift)];
  if (id < 0 || id >= c.pages) {
    report_bad_index(c.status, kTagCachePage);
    return false;
  }
  *page = id;
  return true;
}
// Slots of a sequence's pages, 2^30 at most.
__device__ __forceinline__ int room_of(const Cache4& c) { return c.max_pages << c.page_shift; }
// What the length of sequence b says, none if it is negative.  The status word is set if it is that or more than the pages hold.
__device__ __forceinline__ int length_of(const Cache4& c, int b) {
  const int n = c.lengths[b];
  if (n < 0 || n > room_of(c)) report_bad_index(c.status, kTagCacheLength);
  return max(n, 0);
}
// Tokens of sequence b, no more than its pages hold.
__device__ __forceinline__ int tokens_of(const Cache4& c, int b) { return min(length_of(c, b), room_of(c)); }

}  // namespace
}  // namespace rsfa
