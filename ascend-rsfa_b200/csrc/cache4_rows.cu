// Rows of K and V into a paged cache of 4-bit records and out of it again (the record: ops_common.cuh).
//
// append: per group of 32 dims the minimum m, the scale s = 16-bit((max - min) / 15) and the codes
// rint((x - m) / s) in 0 .. 15; read: s * code + m.  A group whose range is not finite (it holds an infinity or NaN)
// reads back as NaN, one whose scale rounds to nothing as its minimum.
//
// What bounds it: HBM for prompts, the launch for single tokens.  A thread has eight dims, one 16-byte access of the
// dense row, and a row of D dims is D / 8 neighbouring lanes, so a group is four lanes and its range two shuffles.
// Slots run fastest over the warps: neighbouring records of a page are written by neighbouring warps.
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

// Which row a thread has a part of: K (0) or V (1) of row s of head h of sequence b.
struct RowOf {
  int b, h, s, kv, lane;   // lane: which eight dims
};
template <int D>
__device__ __forceinline__ RowOf row_of(long long thread, int H, int S) {
  constexpr int kLanes = D / 8;
  RowOf r;
  r.lane = static_cast<int>(thread % kLanes);
  const long long row = thread / kLanes;
  r.kv = static_cast<int>(row & 1);
  const uint32_t unit = static_cast<uint32_t>(row >> 1);
  const uint32_t bh = unit / S;
  r.s = unit - bh * S;
  r.b = bh / H;
  r.h = bh - r.b * H;
  return r;
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kThreads) cache4_append_kernel(const Cache4 c, const Cache4Rows rows) {
  using R = Record<D>;
  griddep_launch_dependents();
  griddep_wait();
  const long long thread = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  const bool in_range = thread < 2ll * (D / 8) * c.B * c.H * rows.S;
  const RowOf r = row_of<D>(in_range ? thread : 0, c.H, rows.S);
  const int count = rows.counts != nullptr ? min(max(rows.counts[r.b], 0), rows.S) : rows.S;
  const int slot = tokens_of(c, r.b) - count + r.s;
  int64_t page = 0;
  // rows behind the count are padding; a slot below zero is no token (a sequence that is not in use)
  const bool live = in_range && r.s < count && slot >= 0 && find_page(c, r.b, slot, &page);
  float x[8];
  uint4 in = make_uint4(0, 0, 0, 0);
  if (live) {
    const int64_t* st = r.kv ? rows.v_stride : rows.k_stride;
    const uint16_t* src = static_cast<const uint16_t*>(r.kv ? rows.v : rows.k) + r.b * st[0] + r.h * st[1] + r.s * st[2] + 8 * r.lane;
    in = __ldg(reinterpret_cast<const uint4*>(src));
  }
  const uint32_t words[4] = {in.x, in.y, in.z, in.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = to_f32x2<kBf16>(words[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int m = 1; m <= 2; m <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
  }
  if (!live) return;
  const float range = hi - lo;
  const bool finite = range < INFINITY;                       // false for NaN as well
  // The scale is stored in the rows' own type: 11 (8) bits of it are enough for codes of 4 bits, whose
  // rounding is an eighth of a scale and more; the code is chosen for the scale as stored.
  uint16_t s16 = from_f32<kBf16>(range * (1.0f / 15.0f));
  float scale = to_f32<kBf16>(s16);
  if (scale < 1.17549435e-38f) {                              // 1 / scale has to be a number
    scale = 0.f;
    s16 = 0;
  }
  const float inv = scale > 0.f ? __fdiv_rn(1.0f, scale) : 0.f;
  uint32_t codes = 0;
  if (finite) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], lo), inv)), 0.f), 15.f);
      codes |= static_cast<uint32_t>(u) << (4 * i);
    }
  }
  const uint32_t nan16 = kBf16 ? 0x7fc0u : 0x7e00u;
  const uint32_t pair = finite ? (s16 | (static_cast<uint32_t>(from_f32<kBf16>(lo)) << 16)) : (nan16 | (nan16 << 16));
  const int off = slot & ((1 << c.page_shift) - 1);
  uint8_t* rec = c.kv + page * c.kv_stride[0] + r.h * c.kv_stride[1] + static_cast<int64_t>(off) * R::kBytes;
  const int w = r.lane >> 2, q = r.lane & 3;
  if (r.kv == 0) {
    *reinterpret_cast<uint32_t*>(rec + R::k_word(w, q)) = codes;
  } else {
    *reinterpret_cast<uint16_t*>(rec + R::v_half(w, 2 * q)) = static_cast<uint16_t>(codes);
    *reinterpret_cast<uint16_t*>(rec + R::v_half(w, 2 * q + 1)) = static_cast<uint16_t>(codes >> 16);
  }
  if (q == 0) *reinterpret_cast<uint32_t*>(rec + (r.kv ? R::kVPairs : R::kKPairs) + 4 * w) = pair;
  if (r.lane == 0 && r.kv == 0) {
    if (c.weight != nullptr) c.weight[page * c.weight_stride[0] + r.h * c.weight_stride[1] + off] = 0.f;
    if (c.position != nullptr && rows.positions != nullptr)
      c.position[page * c.position_stride[0] + r.h * c.position_stride[1] + off] =
          rows.positions[r.b * rows.positions_stride[0] + r.s * rows.positions_stride[1]];
  }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kThreads) cache4_read_kernel(const Cache4 c, const Cache4Rows rows) {
  using R = Record<D>;
  griddep_launch_dependents();
  griddep_wait();
  const long long thread = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  if (thread >= 2ll * (D / 8) * c.B * c.H * rows.S) return;
  const RowOf r = row_of<D>(thread, c.H, rows.S);
  const long long slot = static_cast<long long>(rows.starts != nullptr ? rows.starts[r.b] : 0) + r.s;
  int64_t page = 0;
  uint4 out = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < tokens_of(c, r.b) && find_page(c, r.b, static_cast<int>(slot), &page)) {
    const int off = static_cast<int>(slot) & ((1 << c.page_shift) - 1);
    const uint8_t* rec = c.kv + page * c.kv_stride[0] + r.h * c.kv_stride[1] + static_cast<int64_t>(off) * R::kBytes;
    const int w = r.lane >> 2, q = r.lane & 3;
    uint32_t codes;
    if (r.kv == 0)
      codes = *reinterpret_cast<const uint32_t*>(rec + R::k_word(w, q));
    else
      codes = *reinterpret_cast<const uint16_t*>(rec + R::v_half(w, 2 * q)) |
              (static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(rec + R::v_half(w, 2 * q + 1))) << 16);
    const float2 sm = to_f32x2<kBf16>(*reinterpret_cast<const uint32_t*>(rec + (r.kv ? R::kVPairs : R::kKPairs) + 4 * w));
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      words[i] = from_f32x2<kBf16>(fmaf(static_cast<float>((codes >> (8 * i)) & 15u), sm.x, sm.y),
                                   fmaf(static_cast<float>((codes >> (8 * i + 4)) & 15u), sm.x, sm.y));
    out = make_uint4(words[0], words[1], words[2], words[3]);
  }
  const int64_t* st = r.kv ? rows.v_stride : rows.k_stride;
  uint16_t* dst = static_cast<uint16_t*>(r.kv ? rows.v : rows.k) + r.b * st[0] + r.h * st[1] + r.s * st[2] + 8 * r.lane;
  *reinterpret_cast<uint4*>(dst) = out;
}

template <typename Kernel>
cudaError_t launch_rows(Kernel kern, const Cache4& c, const Cache4Rows& r, cudaStream_t stream, long long* launches) {
  const long long threads = 2ll * (c.D / 8) * c.B * c.H * r.S;
  const cudaError_t e = launch_persistent(kern, static_cast<int>((threads + kThreads - 1) / kThreads), kThreads, 0, stream,
                                          option_pdl() != 0, c, r);
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
