// Rows of K and V into a paged cache of 4-bit records and out of it again (the record: ops_common.cuh).
//
// append: per group of 32 dims the minimum m, the scale s = 16-bit((max - min) / 15) and the codes
// rint((x - m) / s) in 0 .. 15; read: s * code + m.  A group whose range is not finite (it holds an infinity or NaN)
// reads back as NaN, one whose scale rounds to nothing as its minimum.
//
// What bounds it: HBM for prompts, the launch for single tokens.  A thread has eight dims, one 16-byte access of the
// dense row, and a row of D dims is D / 8 neighbouring lanes, so a group is four lanes and its range two shuffles.
#include "../../include/rsfa.h"
#include "ops_common.cuh"

namespace rsfa {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A CTA has kTokens tokens of one head, two rows of D / 8 lanes each, and a thread the same lane of several of them,
// whose loads go out together: one row at a time, each behind its own lookup of length and page, took twice as long.
constexpr int kTokens = 64;
constexpr int kAtOnce = 4;

struct Chunk {
  int b, h, first, tokens;   // tokens: of this CTA
  int kv, lane, sub, step;   // K (0) or V (1), which eight dims, which token and how many tokens further the next one is
};
template <int D>
__device__ __forceinline__ Chunk chunk_of(const Cache4& c, int S) {
  constexpr int kLanes = D / 8;
  const int chunks = (S + kTokens - 1) / kTokens;
  const int bh = blockIdx.x / chunks;
  Chunk k;
  k.first = (blockIdx.x - bh * chunks) * kTokens;
  k.tokens = min(kTokens, S - k.first);
  k.b = bh / c.H;
  k.h = bh - k.b * c.H;
  k.lane = threadIdx.x % kLanes;
  k.kv = (threadIdx.x / kLanes) & 1;
  k.sub = threadIdx.x / (2 * kLanes);
  k.step = blockDim.x / (2 * kLanes);
  return k;
}

// The V codes of a lane, eight dims of group w, to and from memory order: even groups store the low halves of two
// neighbouring groups, odd ones the high halves.  An exchange that undoes itself.
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
  const Chunk k = chunk_of<D>(c, rows.S);
  // rows behind the count are padding; a slot below zero is no token (a sequence that is not in use)
  const int count = rows.counts != nullptr ? min(max(rows.counts[k.b], 0), rows.S) : rows.S;
  const int slot0 = tokens_of(c, k.b) - count;
  const int64_t* st = k.kv ? rows.v_stride : rows.k_stride;
  const uint16_t* src = static_cast<const uint16_t*>(k.kv ? rows.v : rows.k) + k.b * st[0] + k.h * st[1] + 8 * k.lane;
  const int w = k.lane >> 2, q = k.lane & 3;
  for (int t0 = 0; t0 < k.tokens; t0 += kAtOnce * k.step) {
    uint4 in[kAtOnce];
    int64_t page[kAtOnce];
    bool live[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int t = t0 + i * k.step + k.sub, s = k.first + t;
      live[i] = t < k.tokens && s < count && slot0 + s >= 0 && find_page(c, k.b, slot0 + s, &page[i]);
      in[i] = live[i] ? __ldg(reinterpret_cast<const uint4*>(src + s * st[2])) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int s = k.first + t0 + i * k.step + k.sub;
      const uint32_t words[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = to_f32x2<kBf16>(words[j]);
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
      }
      float lo = x[0], hi = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) {
        lo = min_nan(lo, x[j]);
        hi = max_nan(hi, x[j]);
      }
#pragma unroll
      for (int m = 1; m <= 2; m <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
      }
      const float range = hi - lo;
      const bool finite = range < INFINITY;                       // false for NaN as well
      // The scale is stored in the rows' own type: 11 (8) bits of it are enough for codes of 4 bits, whose
      // rounding is half a scale; the code is chosen for the scale as stored.
      uint16_t s16 = from_f32<kBf16>(range * (1.0f / 15.0f));
      float scale = to_f32<kBf16>(s16);
      if (scale < 1.17549435e-38f) {                              // 1 / scale has to be a number
        scale = 0.f;
        s16 = 0;
      }
      const float inv = scale > 0.f ? __fdiv_rn(1.0f, scale) : 0.f;
      uint32_t codes = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[j], lo), inv)), 0.f), 15.f);   // NaN: 0
        codes |= static_cast<uint32_t>(u) << (4 * j);
      }
      if (!finite) codes = 0;
      const uint32_t turned = exchange_halves<D>(codes, w);
      if (!live[i]) continue;
      const uint32_t nan16 = kBf16 ? 0x7fc0u : 0x7e00u;
      const uint32_t pair = finite ? (s16 | (static_cast<uint32_t>(from_f32<kBf16>(lo)) << 16)) : (nan16 | (nan16 << 16));
      const int off = (slot0 + s) & ((1 << c.page_shift) - 1);
      uint8_t* rec = c.kv + page[i] * c.kv_stride[0] + k.h * c.kv_stride[1] + static_cast<int64_t>(off) * R::kBytes;
      *reinterpret_cast<uint32_t*>(rec + code_word<D>(k.kv, w, q)) = k.kv ? turned : codes;
      if (q == 0) *reinterpret_cast<uint32_t*>(rec + (k.kv ? R::kVPairs : R::kKPairs) + 4 * w) = pair;
      if (k.lane == 0 && k.kv == 0) {
        if (c.weight != nullptr) c.weight[page[i] * c.weight_stride[0] + k.h * c.weight_stride[1] + off] = 0.f;
        if (c.position != nullptr && rows.positions != nullptr)
          c.position[page[i] * c.position_stride[0] + k.h * c.position_stride[1] + off] =
              rows.positions[k.b * rows.positions_stride[0] + s * rows.positions_stride[1]];
      }
    }
  }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kThreads) cache4_read_kernel(const Cache4 c, const Cache4Rows rows) {
  using R = Record<D>;
  griddep_launch_dependents();
  griddep_wait();
  const Chunk k = chunk_of<D>(c, rows.S);
  const long long start = rows.starts != nullptr ? rows.starts[k.b] : 0;
  const int n = tokens_of(c, k.b);
  const int64_t* st = k.kv ? rows.v_stride : rows.k_stride;
  uint16_t* dst = static_cast<uint16_t*>(k.kv ? rows.v : rows.k) + k.b * st[0] + k.h * st[1] + 8 * k.lane;
  const int w = k.lane >> 2, q = k.lane & 3;
  const int at_codes = code_word<D>(k.kv, w, q), at_pair = (k.kv ? R::kVPairs : R::kKPairs) + 4 * w;
  for (int t0 = 0; t0 < k.tokens; t0 += kAtOnce * k.step) {
    uint32_t codes[kAtOnce], pair[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int t = t0 + i * k.step + k.sub;
      const long long slot = start + k.first + t;
      int64_t page;
      codes[i] = pair[i] = 0;
      if (t < k.tokens && slot >= 0 && slot < n && find_page(c, k.b, static_cast<int>(slot), &page)) {
        const uint8_t* rec = c.kv + page * c.kv_stride[0] + k.h * c.kv_stride[1] +
                             (slot & ((1 << c.page_shift) - 1)) * static_cast<int64_t>(R::kBytes);
        codes[i] = *reinterpret_cast<const uint32_t*>(rec + at_codes);
        pair[i] = *reinterpret_cast<const uint32_t*>(rec + at_pair);
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int t = t0 + i * k.step + k.sub;
      const uint32_t turned = exchange_halves<D>(codes[i], w);
      const uint32_t u = k.kv ? turned : codes[i];
      const float2 sm = to_f32x2<kBf16>(pair[i]);
      uint32_t words[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        words[j] = from_f32x2<kBf16>(fmaf(static_cast<float>((u >> (8 * j)) & 15u), sm.x, sm.y),
                                     fmaf(static_cast<float>((u >> (8 * j + 4)) & 15u), sm.x, sm.y));
      if (t < k.tokens) *reinterpret_cast<uint4*>(dst + (k.first + t) * st[2]) = make_uint4(words[0], words[1], words[2], words[3]);
    }
  }
}

template <typename Kernel>
cudaError_t launch_rows(Kernel kern, const Cache4& c, const Cache4Rows& r, cudaStream_t stream, long long* launches) {
  const long long grid = static_cast<long long>(c.B) * c.H * ((r.S + kTokens - 1) / kTokens);
  // a few tokens do not need 256 threads; whole warps, and whole pairs of rows at D = 256
  int threads = (r.S < kTokens ? r.S : kTokens) * 2 * (c.D / 8);
  threads = threads > kThreads ? kThreads : (threads + 31) / 32 * 32;
  const cudaError_t e = launch_persistent(kern, static_cast<int>(grid), threads, 0, stream, option_pdl() != 0, c, r);
  if (e == cudaSuccess) *launches += 1;
  return e;
}

}  // namespace

cudaError_t launch_cache4_append(const Cache4& c, const Cache4Rows& r, cudaStream_t stream, long long* launches) {
  switch (c.D) {
    case 64: return launch_rows(c.bf16 ? cache4_append_kernel<64, true> : cache4_append_kernel<64, false>, c, r, stream, launches);
    case 128: return launch_rows(c.bf16 ? cache4_append_kernel<128, true> : cache4_append_kernel<128, false>, c, r, stream, launches);
    case 256: return launch_rows(c.bf16 ? cache4_append_kernel<256, true> : cache4_append_kernel<256, false>, c, r, stream, launches);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_cache4_read(const Cache4& c, const Cache4Rows& r, cudaStream_t stream, long long* launches) {
  switch (c.D) {
    case 64: return launch_rows(c.bf16 ? cache4_read_kernel<64, true> : cache4_read_kernel<64, false>, c, r, stream, launches);
    case 128: return launch_rows(c.bf16 ? cache4_read_kernel<128, true> : cache4_read_kernel<128, false>, c, r, stream, launches);
    case 256: return launch_rows(c.bf16 ? cache4_read_kernel<256, true> : cache4_read_kernel<256, false>, c, r, stream, launches);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace rsfa
