// Rows of K and V into a paged cache of 4-bit records and out of it again (the record: ops_common.cuh).
//
// append: per group of 32 dims the minimum m, the scale s = 16-bit((max - min) / 15) and the codes
// rint((x - m) / s) in 0 .. 15; read: s * code + m.  A group whose range is not finite (it holds an infinity or NaN)
// reads back as NaN, one whose scale rounds to nothing as its minimum.
//
// What bounds it: HBM for prompts, the launch for single tokens.  A thread that reads has eight dims, one 16-byte access of
// the dense row; one that appends has 16, so that a group is two lanes, its range one shuffle and its scale computed by
// no more than these two (eight: 77 us for 59).  With 8 heads of 128 dims, bf16: 4 sequences of 12288 new tokens are
// appended in 59 us (4.5 TB/s; the instructions of ranges and codes bound it, 76 % of the issue slots; HBM's time is 40), 8
// sequences of up to 4096 tokens, padded, read in 29 us (5.4 TB/s, 77 % of the ALUs), one token of each of 64 sequences appended or
// read in 2.7 us.
#include "../../include/rsfa.h"
#include "ops_common.cuh"

namespace rsfa {
namespace {

constexpr int kThreads = 256;

// Packed minimum and maximum of 16-bit numbers; NaN wins.
template <bool kBf16>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (kBf16)
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (kBf16)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  if constexpr (kBf16)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// Two 32-bit products in one instruction, and a pair of the rows' type less a 32-bit number.
__device__ __forceinline__ float2 times_each(float2 a, float b) {
  float2 r;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %4};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ float2 above(uint32_t pair, float minus_lo) {
  float2 r;
  if constexpr (kBf16)
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\nfma.rn.f32.bf16 %0, l, %3, %4;\nfma.rn.f32.bf16 %1, h, %3, %4;\n}\n"
        : "=f"(r.x), "=f"(r.y) : "r"(pair), "h"(static_cast<uint16_t>(0x3f80)), "f"(minus_lo));
  else
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\nfma.rn.f32.f16 %0, l, %3, %4;\nfma.rn.f32.f16 %1, h, %3, %4;\n}\n"
        : "=f"(r.x), "=f"(r.y) : "r"(pair), "h"(static_cast<uint16_t>(0x3c00)), "f"(minus_lo));
  return r;
}
// Codes 2 j and 2 j + 1 of a word as a pair of 16-bit numbers: put where the mantissa of 1024 (fp16) or 128 (bf16) ends,
// which then comes off exactly.  (An integer conversion per code is four times as slow as all the rest.)
template <bool kBf16>
__device__ __forceinline__ uint32_t code_pair(uint32_t codes, int j) {
  const uint32_t both = __byte_perm(codes, 0u, 0x4040 + 0x0101 * j);   // byte j in either half
  if constexpr (kBf16) return fma2<true>((both & 0x0000000fu) | ((both >> 4) & 0x000f0000u) | 0x43004300u, 0x3f803f80u, 0xc300c300u);
  // the second code stands four bits higher: 1024 + 16 u
  return fma2<false>((both & 0x00f0000fu) | 0x64006400u, 0x2c003c00u, 0xd400e400u);
}

// A CTA has kTokens tokens of one head, two rows of D / kReadDims or D / kAppendDims lanes each, and a thread the same lane
// of several of them, whose loads go out together: one row at a time, each behind its own lookup of length and page, took
// twice as long.
constexpr int kTokens = 64;
constexpr int kReadDims = 8, kAppendDims = 16;
constexpr int kAtOnce = 4;
constexpr int kAppendAtOnce = 1;   // and as many on their way (two: 67 us for 59 below, in 78 registers for 48)

struct Chunk {
  int b, h, first, tokens;   // tokens: of this CTA
  int kv, lane, sub, step;   // K (0) or V (1), which dims, which token and how many tokens further the next one is
};
template <int kLanes>
__device__ __forceinline__ Chunk chunk_of(const Cache4& c, int S) {
  const int chunks = (S + kTokens - 1) / kTokens;
  Chunk k;
  // heads first: in a [B, S, H, D] projection their rows of a token lie side by side
  const int bc = blockIdx.x / c.H;
  k.h = blockIdx.x - bc * c.H;
  k.b = bc / chunks;
  k.first = (bc - k.b * chunks) * kTokens;
  k.tokens = min(kTokens, S - k.first);
  k.lane = threadIdx.x % kLanes;
  k.kv = (threadIdx.x / kLanes) & 1;
  k.sub = threadIdx.x / (2 * kLanes);
  k.step = blockDim.x / (2 * kLanes);
  return k;
}

// The pages that slots first .. first + kTokens - 1 of a sequence lie in, looked up once for all rows of the CTA.
constexpr int kChunkPages = kTokens / 16 + 1;
struct ChunkPages {
  int64_t page[kChunkPages];       // -1: none
  int64_t records[kChunkPages];    // bytes from the start of the cache, for the CTA's head
  int missing;                     // whether any is none
};
__device__ __forceinline__ void find_pages(ChunkPages& at, const Cache4& c, const Chunk& k, int first, int end) {
  if (threadIdx.x == 0) at.missing = 0;
  __syncwarp();                    // the first warp has all of them
  if (threadIdx.x < kChunkPages) {
    const int slot = ((first >> c.page_shift) + static_cast<int>(threadIdx.x)) << c.page_shift;   // the first of the page
    int64_t page = -1;
    if (slot >= end || !find_page(c, k.b, slot, &page)) page = -1;
    if (slot < end && page < 0) at.missing = 1;
    at.page[threadIdx.x] = page;
    at.records[threadIdx.x] = (page < 0 ? 0 : page) * c.kv_stride[0] + k.h * c.kv_stride[1];
  }
  __syncthreads();
}

// The V codes of a reading lane, eight dims of group w, from memory order: even groups have the low halves of two
// neighbouring groups, odd ones the high halves.
template <int D>
__device__ __forceinline__ uint32_t exchange_halves(uint32_t codes, int w) {
  const uint32_t other = __shfl_xor_sync(0xffffffffu, codes, 4);
  return (w & 1) ? __byte_perm(other, codes, 0x7632) : __byte_perm(codes, other, 0x5410);
}
// Where that word is: K word (w, q), or the V half words (w, w + 1) of chunk 2 q (even w) or 2 q + 1 (odd w).
template <int D>
__device__ __forceinline__ int code_word(int kv, int w, int q) {
  using R = Record<D>;
  return kv == 0 ? R::k_word(w, q) : R::v_half(w & ~1, 2 * q + (w & 1));
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kThreads) cache4_append_kernel(const Cache4 c, const Cache4Rows rows) {
  using R = Record<D>;
  griddep_launch_dependents();
  griddep_wait();
  const Chunk k = chunk_of<D / kAppendDims>(c, rows.S);
  // rows behind the count are padding; a slot below zero is no token (a sequence that is not in use)
  const int count = rows.counts != nullptr ? min(max(rows.counts[k.b], 0), rows.S) : rows.S;
  int to = min(k.tokens, count - k.first);
  if (to <= 0) return;
  // The first rows are asked for before the sequence's length and pages are.
  const int64_t* st = k.kv ? rows.v_stride : rows.k_stride;
  const int64_t step_bytes = st[2] * 2 * k.step;
  const uint8_t* src = static_cast<const uint8_t*>(k.kv ? rows.v : rows.k) + 2 * (k.b * st[0] + k.h * st[1] + kAppendDims * k.lane + (k.first + k.sub) * st[2]);
  uint4 next[kAppendAtOnce][2];
  auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < kAppendAtOnce; ++i) {
      const bool any = t0 + i * k.step + k.sub < to;
#pragma unroll
      for (int j = 0; j < 2; ++j) next[i][j] = any ? reinterpret_cast<const uint4*>(src)[j] : make_uint4(0, 0, 0, 0);
      src += step_bytes;
    }
  };
  load(0);
  const int slot0 = length_of(c, k.b) - count + k.first;       // of the CTA's first token
  // of a length beyond the pages the rows behind them are left out, not put in the place of others
  to = static_cast<int>(min(static_cast<long long>(to), static_cast<long long>(room_of(c)) - slot0));
  const int from = max(0, -slot0);
  if (from >= to) return;
  __shared__ ChunkPages at;
  const int page0 = (slot0 + from) >> c.page_shift;
  find_pages(at, c, k, slot0 + from, slot0 + to);
  // The lane's dims are words 2 j and 2 j + 1 of group w.  It stores both of K; of V, whose memory words have four dims of
  // an even group and of the odd one behind it, the lane of the even group stores what has word 2 j of either and
  // that of the odd one what has word 2 j + 1.
  const int w = k.lane >> 1, j = k.lane & 1;
  const bool odd = (w & 1) != 0;
  const int at_codes = k.kv ? R::v_half(w & ~1, 4 * j + 2 * (w & 1)) : R::k_word(w, 2 * j);
  const int at_second = k.kv ? R::v_half(0, 1) - R::v_half(0, 0) : R::k_word(0, 1) - R::k_word(0, 0);
  const int at_pair = (k.kv ? R::kVPairs : R::kKPairs) + 4 * w;
  const int mask = (1 << c.page_shift) - 1;
  const bool missing = at.missing != 0;
  uint8_t* const kv_codes = c.kv + at_codes;
  for (int t0 = 0; t0 < to; t0 += kAppendAtOnce * k.step) {
    uint4 in[kAppendAtOnce][2];
    bool live[kAppendAtOnce];
#pragma unroll
    for (int i = 0; i < kAppendAtOnce; ++i) {
      const int t = t0 + i * k.step + k.sub;
      in[i][0] = next[i][0];
      in[i][1] = next[i][1];
      live[i] = t >= from && t < to && !(missing && at.page[((slot0 + t) >> c.page_shift) - page0] < 0);
    }
    if (t0 + kAppendAtOnce * k.step < to) load(t0 + kAppendAtOnce * k.step);
#pragma unroll
    for (int i = 0; i < kAppendAtOnce; ++i) {
      const int slot = slot0 + t0 + i * k.step + k.sub;
      const uint32_t words[8] = {in[i][0].x, in[i][0].y, in[i][0].z, in[i][0].w, in[i][1].x, in[i][1].y, in[i][1].z, in[i][1].w};
      uint32_t lo2 = words[0], hi2 = words[0];
#pragma unroll
      for (int m = 1; m < 8; ++m) {
        lo2 = min2<kBf16>(lo2, words[m]);
        hi2 = max2<kBf16>(hi2, words[m]);
      }
      // the smaller of each half in the low half, the larger in the high one
      uint32_t ends = __byte_perm(min2<kBf16>(lo2, lo2 >> 16), max2<kBf16>(hi2, hi2 >> 16), 0x5410);
      const uint32_t others = __shfl_xor_sync(0xffffffffu, ends, 1);
      ends = __byte_perm(min2<kBf16>(ends, others), max2<kBf16>(ends, others), 0x7610);
      const float2 range2 = to_f32x2<kBf16>(ends);
      const float lo = range2.x, range = range2.y - range2.x;
      const bool finite = range < INFINITY;                       // false for NaN as well
      // The scale is stored in the rows' own type: 11 (8) bits of it are enough for codes of 4 bits, whose
      // rounding is half a scale; the code is chosen for the scale as stored.
      uint16_t s16 = from_f32<kBf16>(range * (1.0f / 15.0f));
      float scale = to_f32<kBf16>(s16);
      if (scale < 1.17549435e-38f) {                              // 1 / scale has to be a number
        scale = 0.f;
        s16 = 0;
      }
      const float inv = scale > 0.f ? __frcp_rn(scale) : 0.f;
      // (x - lo) / scale is rounded to an integer by the sum with 1.5 * 2^23, whose low bits it then is; those of the
      // eight sums, each four bits further up, make the word, and what 1.5 * 2^23 adds to it is one constant.
      // A quotient is above 15.5 only where the scale is one of fp16's subnormal numbers: a normal one, and every one of
      // bf16 that is not taken for zero, is 2^-8 of itself below range / 15 at most.
      uint32_t codes[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        codes[half] = 0;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          float2 x = times_each(above<kBf16>(words[4 * half + m], -lo), inv);
          if constexpr (!kBf16) x = make_float2(fminf(x.x, 15.f), fminf(x.y, 15.f));
          codes[half] += (__float_as_uint(__fadd_rn(x.x, 12582912.f)) << (8 * m)) + (__float_as_uint(__fadd_rn(x.y, 12582912.f)) << (8 * m + 4));
        }
        codes[half] -= 0x4b400000u * 0x11111111u;
        if (!finite) codes[half] = 0;
      }
      const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? codes[0] : codes[1], 2);
      if (k.kv) {
        const uint32_t even_codes = odd ? other : codes[0], odd_codes = odd ? codes[1] : other;
        codes[0] = __byte_perm(even_codes, odd_codes, 0x5410);
        codes[1] = __byte_perm(even_codes, odd_codes, 0x7632);
      }
      if (!live[i]) continue;
      const uint32_t nan16 = kBf16 ? 0x7fc0u : 0x7e00u;
      const uint32_t pair = finite ? (s16 | (ends << 16)) : (nan16 | (nan16 << 16));
      const int off = slot & mask, which = (slot >> c.page_shift) - page0;
      uint8_t* rec = kv_codes + (at.records[which] + off * R::kBytes);
      *reinterpret_cast<uint32_t*>(rec) = codes[0];
      *reinterpret_cast<uint32_t*>(rec + at_second) = codes[1];
      if (j == 0) *reinterpret_cast<uint32_t*>(rec + (at_pair - at_codes)) = pair;
    }
  }
  // what else there is of the tokens, one per thread
  for (int t = from + threadIdx.x; t < to; t += blockDim.x) {
    const int slot = slot0 + t;
    const int64_t page = at.page[(slot >> c.page_shift) - page0];
    if (page < 0) continue;
    if (c.weight != nullptr) c.weight[page * c.weight_stride[0] + k.h * c.weight_stride[1] + (slot & mask)] = 0.f;
    if (c.position != nullptr && rows.positions != nullptr)
      c.position[page * c.position_stride[0] + k.h * c.position_stride[1] + (slot & mask)] =
          rows.positions[k.b * rows.positions_stride[0] + (k.first + t) * rows.positions_stride[1]];
  }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kThreads) cache4_read_kernel(const Cache4 c, const Cache4Rows rows) {
  using R = Record<D>;
  griddep_launch_dependents();
  griddep_wait();
  const Chunk k = chunk_of<D / kReadDims>(c, rows.S);
  // slots of the CTA's tokens: `from` to `to` are in use, the others read as zeros
  const long long slot0 = static_cast<long long>(rows.starts != nullptr ? rows.starts[k.b] : 0) + k.first;
  const int n = tokens_of(c, k.b);
  const int from = static_cast<int>(min(static_cast<long long>(k.tokens), max(0ll, -slot0)));
  const int to = static_cast<int>(max(static_cast<long long>(from), min(static_cast<long long>(k.tokens), n - slot0)));
  __shared__ ChunkPages at;
  const int first = from < to ? static_cast<int>(slot0 + from) : 0, page0 = first >> c.page_shift;
  find_pages(at, c, k, first, first + to - from);
  const int64_t* st = k.kv ? rows.v_stride : rows.k_stride;
  const int64_t step_bytes = st[2] * 2 * k.step;
  uint8_t* dst = static_cast<uint8_t*>(k.kv ? rows.v : rows.k) + 2 * (k.b * st[0] + k.h * st[1] + 8 * k.lane + (k.first + k.sub) * st[2]);
  const int w = k.lane >> 2, q = k.lane & 3;
  const int at_codes = code_word<D>(k.kv, w, q), at_pair = (k.kv ? R::kVPairs : R::kKPairs) + 4 * w;
  const int mask = (1 << c.page_shift) - 1;
  const bool missing = at.missing != 0;
  for (int t0 = 0; t0 < k.tokens; t0 += kAtOnce * k.step) {
    uint32_t codes[kAtOnce], pair[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int t = t0 + i * k.step + k.sub;
      codes[i] = pair[i] = 0;
      if (t >= from && t < to) {
        const int slot = first + t - from, which = (slot >> c.page_shift) - page0;
        if (!(missing && at.page[which] < 0)) {
          const uint8_t* rec = c.kv + (at.records[which] + (slot & mask) * R::kBytes);
          codes[i] = *reinterpret_cast<const uint32_t*>(rec + at_codes);
          pair[i] = *reinterpret_cast<const uint32_t*>(rec + at_pair);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int t = t0 + i * k.step + k.sub;
      const uint32_t turned = exchange_halves<D>(codes[i], w);
      const uint32_t u = k.kv ? turned : codes[i];
      // one rounding, to the rows' type
      const uint32_t scales = __byte_perm(pair[i], pair[i], 0x1010), minima = __byte_perm(pair[i], pair[i], 0x3232);
      uint32_t words[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) words[j] = fma2<kBf16>(code_pair<kBf16>(u, j), scales, minima);
      if (t < k.tokens) *reinterpret_cast<uint4*>(dst) = make_uint4(words[0], words[1], words[2], words[3]);
      dst += step_bytes;
    }
  }
}

template <typename Kernel>
cudaError_t launch_rows(Kernel kern, int dims, const Cache4& c, const Cache4Rows& r, cudaStream_t stream, long long* launches) {
  const long long grid = static_cast<long long>(c.B) * c.H * ((r.S + kTokens - 1) / kTokens);
  // a few tokens do not need 256 threads; whole warps
  int threads = (r.S < kTokens ? r.S : kTokens) * 2 * (c.D / dims);
  threads = threads > kThreads ? kThreads : (threads + 31) / 32 * 32;
  const cudaError_t e = launch_persistent(kern, static_cast<int>(grid), threads, 0, stream, option_pdl() != 0, c, r);
  if (e == cudaSuccess) *launches += 1;
  return e;
}

}  // namespace

cudaError_t launch_cache4_append(const Cache4& c, const Cache4Rows& r, cudaStream_t stream, long long* launches) {
  switch (c.D) {
    case 64: return launch_rows(c.bf16 ? cache4_append_kernel<64, true> : cache4_append_kernel<64, false>, kAppendDims, c, r, stream, launches);
    case 128: return launch_rows(c.bf16 ? cache4_append_kernel<128, true> : cache4_append_kernel<128, false>, kAppendDims, c, r, stream, launches);
    case 256: return launch_rows(c.bf16 ? cache4_append_kernel<256, true> : cache4_append_kernel<256, false>, kAppendDims, c, r, stream, launches);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_cache4_read(const Cache4& c, const Cache4Rows& r, cudaStream_t stream, long long* launches) {
  switch (c.D) {
    case 64: return launch_rows(c.bf16 ? cache4_read_kernel<64, true> : cache4_read_kernel<64, false>, kReadDims, c, r, stream, launches);
    case 128: return launch_rows(c.bf16 ? cache4_read_kernel<128, true> : cache4_read_kernel<128, false>, kReadDims, c, r, stream, launches);
    case 256: return launch_rows(c.bf16 ? cache4_read_kernel<256, true> : cache4_read_kernel<256, false>, kReadDims, c, r, stream, launches);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace rsfa
