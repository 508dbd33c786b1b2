// Rotary positions for B200 (sm_100a): q and k turned by their positions in one launch, and the table of
// cosines and sines that they are turned by.
//
// The pair (a, b) of frequency i at position p becomes (a c - b s, b c + a s) with (c, s) = table[p][i]; the
// gradient is the transposed rotation, the same kernel with s negated (`inverse`).  A pair is (2 i, 2 i + 1) in the
// interleaved layout and (i, i + R / 2) in the half layout; dims from R on are copied.
//
// What bounds it: HBM, q and k read once and written once.  A thread owns the same 16 bytes of columns (half
// layout: 16 bytes of each half) of several heads of one position, so that the table entries, twice the bytes of
// the data they turn, are read once for all of these heads.  16 sequences of 4096 positions, 16 + 16 heads of 128 dims,
// bf16: 163.2 us, 6.6 TB/s, what a plain copy of these bytes takes; 8 of 1000, 32 + 8 heads, 64 of 128 dims turned: 28.0 us
// interleaved and 30.0 in halves (5.8 and 5.5 TB/s).  Where the dims that turn are no multiple of 16 (8 interleaved), a thread has
// one pair in accesses of two bytes: 8, 20, 24 or 30 of the 128 dims in halves 70 us, 20 or 30 interleaved 63.  The table of
// 131072 positions by 64 frequencies, 67 MB, takes 13.3 us (5.1 TB/s): its sines and cosines, one pair per 8 bytes, are about as
// long as their stores.
#include "../../include/rsfa.h"
#include "ops_common.cuh"

namespace rsfa {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ long long position_of(const RotaryParams& p, int b, int s) {
  if (p.positions == nullptr) return s;
  const int64_t at = b * p.pos_stride[0] + s * p.pos_stride[1];
  return p.positions_64 ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
}

template <bool kBf16>
__device__ __forceinline__ void turn_halves(uint4& a, uint4& b, const float2 (&cs)[8]) {
  uint32_t* pa = reinterpret_cast<uint32_t*>(&a);
  uint32_t* pb = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = to_f32x2<kBf16>(pa[i]), y = to_f32x2<kBf16>(pb[i]);
    const float2 t = cs[2 * i], u = cs[2 * i + 1];
    pa[i] = from_f32x2<kBf16>(x.x * t.x - y.x * t.y, x.y * u.x - y.y * u.y);
    pb[i] = from_f32x2<kBf16>(y.x * t.x + x.x * t.y, y.y * u.x + x.y * u.y);
  }
}
template <bool kBf16>
__device__ __forceinline__ void turn_pairs(uint4& a, const float2 (&cs)[8]) {
  uint32_t* pa = reinterpret_cast<uint32_t*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = to_f32x2<kBf16>(pa[i]);
    pa[i] = from_f32x2<kBf16>(x.x * cs[i].x - x.y * cs[i].y, x.y * cs[i].x + x.x * cs[i].y);
  }
}

// kWide: 16 bytes at a time (R a multiple of 16 in the half layout, of 8 interleaved).  Otherwise a thread owns
// one pair, or two neighbouring columns behind R.
template <bool kBf16, bool kInterleaved, bool kWide>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p, const int chunks, const int turned, const int heads_each) {
  griddep_launch_dependents();
  griddep_wait();
  const uint32_t unit = blockIdx.x * kThreads + threadIdx.x;
  if (unit >= static_cast<uint32_t>(p.B) * p.S * chunks) return;
  const int row = unit / chunks, chunk = unit - row * chunks;
  const int b = row / p.S, s = row - b * p.S;
  const bool turns = chunk < turned;
  const long long pos = position_of(p, b, s);
  const bool known = pos >= 0 && pos < p.table_length;
  if (!known && chunk == 0 && blockIdx.y == 0) report_bad_index(p.status, kTagRotaryPosition);
  const float2* table = reinterpret_cast<const float2*>(p.table) + (known ? pos : 0) * (p.R >> 1);
  const float sign = p.inverse ? -1.f : 1.f;
  const float lost = known ? 0.f : __int_as_float(0x7fffffff);   // a row without a position comes out as NaN,
  const uint32_t lost16 = known ? 0u : 0x7fff7fffu;               // in either type, where it is copied as well

  constexpr int kPairs = kWide ? (kInterleaved ? 4 : 8) : 1;
  float2 cs[8];
  if (turns) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 t = table[chunk * kPairs + i];
      cs[i] = make_float2(t.x + lost, t.y * sign);
    }
  }
  const int half = p.R >> 1;
  const int h0 = blockIdx.y * heads_each;
  const int h1 = min(h0 + heads_each, p.heads[0] + p.heads[1]);
  // column of the thread's (first) data; the half layout's partner lies R / 2 further
  int col;
  if constexpr (kWide)
    col = turns ? chunk * 8 : p.R + (chunk - turned) * 8;
  else
    col = turns ? (kInterleaved ? 2 * chunk : chunk) : p.R + (chunk - turned) * 2;

  auto address = [&](int h, const uint16_t** src, uint16_t** dst) {
    const int t = h >= p.heads[0];
    const int64_t hh = t ? h - p.heads[0] : h;
    *src = static_cast<const uint16_t*>(p.x[t]) + b * p.x_stride[t][0] + hh * p.x_stride[t][1] + s * p.x_stride[t][2] + col;
    *dst = static_cast<uint16_t*>(p.y[t]) + b * p.y_stride[t][0] + hh * p.y_stride[t][1] + s * p.y_stride[t][2] + col;
  };
  if constexpr (kWide) {
    constexpr int kAtOnce = kInterleaved ? 8 : 4;   // heads whose loads go out together
    for (int h = h0; h < h1; h += kAtOnce) {
      uint4 a[kAtOnce], c[kAtOnce];
      uint16_t* dst[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (h + i < h1) {
          const uint16_t* src;
          address(h + i, &src, &dst[i]);
          a[i] = *reinterpret_cast<const uint4*>(src);
          if (!kInterleaved && turns) c[i] = *reinterpret_cast<const uint4*>(src + half);
        }
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (h + i < h1) {
          if (turns) {
            if constexpr (kInterleaved) {
              turn_pairs<kBf16>(a[i], cs);
            } else {
              turn_halves<kBf16>(a[i], c[i], cs);
              *reinterpret_cast<uint4*>(dst[i] + half) = c[i];
            }
          }
          if (!turns) a[i].x |= lost16, a[i].y |= lost16, a[i].z |= lost16, a[i].w |= lost16;
          *reinterpret_cast<uint4*>(dst[i]) = a[i];
        }
      }
    }
  } else {
    for (int h = h0; h < h1; ++h) {
      const uint16_t* src;
      uint16_t* dst;
      address(h, &src, &dst);
      const int other = (turns && !kInterleaved) ? half : 1;
      uint16_t a = src[0], c = src[other];
      if (turns) {
        const float x = to_f32<kBf16>(a), y = to_f32<kBf16>(c);
        a = from_f32<kBf16>(x * cs[0].x - y * cs[0].y);
        c = from_f32<kBf16>(y * cs[0].x + x * cs[0].y);
      } else {
        a |= lost16;
        c |= lost16;
      }
      dst[0] = a;
      dst[other] = c;
    }
  }
}

template <bool kBf16, bool kInterleaved, bool kWide>
cudaError_t launch_one(const RotaryParams& p, int sm_count, cudaStream_t stream, long long* launches) {
  const int per = kWide ? 8 : 2;                                        // columns of a chunk that is copied
  const int turned = kWide ? p.R / (kInterleaved ? 8 : 16) : p.R / 2;
  const int chunks = turned + (p.D - p.R) / per;
  const long long blocks = (static_cast<long long>(p.B) * p.S * chunks + kThreads - 1) / kThreads;
  const int heads = p.heads[0] + p.heads[1];
  // As many heads per thread as leave every multiprocessor a few CTAs: they share the table's entries.
  int each = 16;
  while (each > 1 && blocks * ((heads + each - 1) / each) < 4ll * sm_count) each >>= 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), static_cast<unsigned>((heads + each - 1) / each));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option_pdl() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, rotary_kernel<kBf16, kInterleaved, kWide>, p, chunks, turned, each);
  if (e == cudaSuccess) *launches += 1;
  return e;
}

// ------------------------------------------------------------------ the table
struct TableArgs {
  double base, factor, original, low, high, multiplier;
  int scaling, length, dim;
};

constexpr int kTableRows = 64;   // positions per thread

// The angle per position of frequency i, scaled for long contexts.
__device__ double frequency(const TableArgs& t, int i) {
  double base = t.base;
  if (t.scaling == RSFA_ROTARY_NTK && t.dim > 2) base *= pow(t.factor, t.dim / (t.dim - 2.0));
  const double f = pow(base, -2.0 * i / t.dim);
  if (t.scaling == RSFA_ROTARY_LINEAR || (t.scaling == RSFA_ROTARY_NTK && t.dim == 2)) return f / t.factor;
  const double kTurn = 6.283185307179586476925286766559;
  if (t.scaling == RSFA_ROTARY_YARN) {
    // the pair whose angle makes `turns` turns over the original length
    const double at_high = t.dim * log(t.original / (kTurn * t.high)) / (2.0 * log(t.base));
    const double at_low = t.dim * log(t.original / (kTurn * t.low)) / (2.0 * log(t.base));
    const double lo = fmax(floor(at_high), 0.0), hi = fmin(ceil(at_low), t.dim - 1.0);
    const double ramp = fmin(fmax((i - lo) / fmax(hi - lo, 0.001), 0.0), 1.0);
    return f * (1.0 - ramp) + f / t.factor * ramp;
  }
  if (t.scaling == RSFA_ROTARY_BANDS) {
    const double share = fmin(fmax((t.original * f / kTurn - t.low) / (t.high - t.low), 0.0), 1.0);
    return f * share + f / t.factor * (1.0 - share);
  }
  return f;
}

// One thread: kTableRows positions of one frequency.  The first angle goes through sincospi, the others follow by
// turning in 64 bits: an error of 64 roundings of 2^-53 each, nothing next to the entries' 2^-24.  The powers that a frequency
// takes are worked out once per CTA; with one per thread they took as long as the table's way to memory.
__global__ void __launch_bounds__(kThreads) rotary_table_kernel(float2* table, const TableArgs t) {
  __shared__ double turns[128];            // per position, in halves
  const int half = t.dim >> 1;
  for (int i = threadIdx.x; i < half; i += kThreads) turns[i] = frequency(t, i) * 0.31830988618379067153776752674503;
  __syncthreads();
  griddep_launch_dependents();
  griddep_wait();
  const long long unit = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  const int block = static_cast<int>(unit / half), i = static_cast<int>(unit - static_cast<long long>(block) * half);
  const long long first = static_cast<long long>(block) * kTableRows;
  if (first >= t.length) return;
  const double f = turns[i];
  double s, c, ds, dc;
  sincospi(static_cast<double>(first) * f, &s, &c);
  sincospi(f, &ds, &dc);
  s *= t.multiplier;
  c *= t.multiplier;
  const int rows = static_cast<int>(min(static_cast<long long>(kTableRows), t.length - first));
  float2* out = table + first * half + i;
  for (int r = 0; r < rows; ++r) {
    *out = make_float2(static_cast<float>(c), static_cast<float>(s));
    out += half;
    const double n = c * dc - s * ds;
    s = s * dc + c * ds;
    c = n;
  }
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, int sm_count, cudaStream_t stream, long long* launches) {
  const bool wide = p.R % (p.interleaved ? 8 : 16) == 0;
  if (p.bf16) {
    if (p.interleaved)
      return wide ? launch_one<true, true, true>(p, sm_count, stream, launches) : launch_one<true, true, false>(p, sm_count, stream, launches);
    return wide ? launch_one<true, false, true>(p, sm_count, stream, launches) : launch_one<true, false, false>(p, sm_count, stream, launches);
  }
  if (p.interleaved)
    return wide ? launch_one<false, true, true>(p, sm_count, stream, launches) : launch_one<false, true, false>(p, sm_count, stream, launches);
  return wide ? launch_one<false, false, true>(p, sm_count, stream, launches) : launch_one<false, false, false>(p, sm_count, stream, launches);
}

cudaError_t launch_rotary_table(float* table, int length, int dim, const double* a, int scaling, cudaStream_t stream,
                                long long* launches) {
  const TableArgs t = {a[0], a[1], a[2], a[3], a[4], a[5], scaling, length, dim};
  const long long units = (static_cast<long long>(length) + kTableRows - 1) / kTableRows * (dim / 2);
  const cudaError_t e = launch_persistent(rotary_table_kernel, static_cast<int>((units + kThreads - 1) / kThreads), kThreads, 0, stream,
                                          option_pdl() != 0, reinterpret_cast<float2*>(table), t);
  if (e == cudaSuccess) *launches += 1;
  return e;
}

}  // namespace rsfa
