// Attention of a few query tokens per sequence over a paged cache of 4-bit records (the record: ops_common.cuh).
//
// With codes u, scales s and minima m per token t and group g of 32 dims,
//   score(t) = sm_scale * sum_g [ s_g(t) * sum_{d in g} q_d u_d(t)  +  m_g(t) * sum_{d in g} q_d ]
//   O_d      = sum_t p(t) s_g(t) u_d(t)  +  sum_t p(t) m_g(t),          p = softmax over the visible tokens
// so the products run over the codes themselves and no value is ever written out.  Both are warp-level MMAs with the
// cache as the A operand (rows are tokens, then dims) and up to 8 query rows as the B operand: the query heads
// that share a K/V head, times the query tokens.  A code needs no conversion: four bits at the bottom of a 16-bit
// word ARE the fp16 number u * 2^-24, one position further up u * 2^-20, and MMAs take subnormal operands as they are;
// the powers of two come out in the scores' factor and in the accumulators' final one.
//
// Rows of scores are handed on by a flash recurrence whose reference is raised only when a score exceeds it by 8
// log2 units.  p * s is rounded to fp16 for the second product; p, its sum and the minima's term stay in 32 bits.
//
// What bounds it: HBM, 5 D / 4 bytes per token and K/V head, and close behind it the instructions that take the codes
// apart.  The work is the list of all tiles of 32 tokens of all (sequence, K/V head, block of query rows), and every warp of
// the device takes an equal, contiguous share of it, whatever the lengths are.  A share's first and last item may
// continue in other warps: their sums go to a workspace and a second kernel joins them.
#include "../../include/rsfa.h"
#include "ops_common.cuh"

namespace rsfa {
namespace {

constexpr int kTile = 32;            // tokens per tile
constexpr int kWarps = 4;            // per CTA
constexpr int kThreads = 32 * kWarps;
constexpr int kJoinThreads = 128;
#ifndef C4_CTAS128
#define C4_CTAS128 4
#define C4_STAGES128 2
#endif
// CTAs per multiprocessor by the registers of their accumulators, and slots of a warp's ring by its shared memory.
template <int D, int NT>
struct Shape {
  static constexpr int kCtas = D == 256 ? 2 : NT == 2 ? (D == 64 ? 3 : 2) : C4_CTAS128;
  static constexpr int kStages = D == 64 ? 4 : D == 256 ? 2 : NT == 2 ? 4 : C4_STAGES128;
  static constexpr int kSlotBytes = kTile * Record<D>::kBytes;
  static constexpr int kRingBytes = kWarps * kStages * kSlotBytes;
};
constexpr int kTagCache4Load = 40;   // of a bounded wait, in the status word
constexpr float kRaise = 8.f;        // log2 units above the reference at which it is raised
constexpr float kRaiseScale = 64.f;  // and the scales' one

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Global to this CTA's shared memory, both 16-byte aligned, counted in bytes on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bar, uint32_t bytes) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// ------------------------------------------------------------------ the list of tiles
// Items are (sequence, K/V head, block of query rows) in this order, an item's tiles follow one another.
struct Items {
  int per_sequence;    // K/V heads * blocks of rows
  long long total;     // tiles
};
__device__ __forceinline__ int visible_tokens(const Cache4& c, const int* counts, int b) {
  return counts != nullptr && counts[b] <= 0 ? 0 : tokens_of(c, b);
}
__device__ __forceinline__ int tiles_of(const Cache4& c, const int* counts, int b) {
  return (visible_tokens(c, counts, b) + kTile - 1) / kTile;
}
// One warp: tiles of the sequences below `end`, per item.
__device__ __forceinline__ long long tiles_before(const Cache4& c, const int* counts, int end) {
  long long n = 0;
  for (int b = threadIdx.x & 31; b < end; b += 32) n += tiles_of(c, counts, b);
#pragma unroll
  for (int d = 16; d; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
  return n;
}
// One warp: the sequence that tile `at` belongs to and the first tile of that sequence.
__device__ __forceinline__ int sequence_of(const Cache4& c, const int* counts, int per_sequence, long long at, long long* first, int* tiles) {
  const int lane = threadIdx.x & 31;
  long long before = 0;
  for (int base = 0; base < c.B; base += 32) {
    const int mine = base + lane < c.B ? tiles_of(c, counts, base + lane) : 0;
    long long sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += u;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, (before + sum) * per_sequence > at);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      *tiles = __shfl_sync(0xffffffffu, mine, l);
      *first = (before + __shfl_sync(0xffffffffu, sum, l) - *tiles) * per_sequence;
      return base + l;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return -1;
}
// Worker w of `workers`, no more than there are tiles, has the tiles from share_begin(w) to share_begin(w + 1).  Its number
// goes over the CTAs first, so that a few tiles are spread over all multiprocessors.
__device__ __forceinline__ long long worker_here() { return static_cast<long long>(threadIdx.x >> 5) * gridDim.x + blockIdx.x; }
__device__ __forceinline__ long long workers_used(long long total, long long all) { return total < all ? total : all; }
__device__ __forceinline__ long long share_begin(long long total, long long worker, long long workers) {
  return total * worker / workers;
}
__device__ __forceinline__ long long worker_of(long long total, long long tile, long long workers) {
  return ((tile + 1) * workers - 1) / total;
}

// ------------------------------------------------------------------ query rows
// Row r of an item is query token r / group of head (r % group) of the K/V head's query heads.
struct Rows {
  int group, count;    // query heads per K/V head; rows = group * S
};

// The B fragments of 8 NT query rows, each row divided by a power of two so that its largest element is about 2^10
// (fp16 then holds bf16's numbers as well), the sums of its groups and its factor.
template <int D, int NT>
struct Query {
  static constexpr int G = D / 32;
  uint32_t frag[NT][G][4];
  float sums[NT][G][2];     // of rows 2 c, 2 c + 1 (c = lane % 4), times 2^-24
  float factor[NT][2];
  int last[NT][2];          // last visible slot
};

template <int D, int NT, bool kBf16>
__device__ __forceinline__ void load_query(Query<D, NT>& f, const Cache4& c, const Cache4Attention& a, const Rows& rows, int b, int h, int row0, int n) {
  constexpr int G = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int count = a.counts != nullptr ? min(a.counts[b], a.S) : a.S;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = row0 + 8 * nt + g;
    float x[G][8];
    float top = 0.f;
    if (row < rows.count) {
      const int i = row / rows.group, hq = h * rows.group + row - i * rows.group;
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + hq * a.q_stride[1] + i * a.q_stride[2] + 8 * q4;
#pragma unroll
      for (int w = 0; w < G; ++w) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + 32 * w));
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 t = to_f32x2<kBf16>(words[j]);
          x[w][2 * j] = t.x;
          x[w][2 * j + 1] = t.y;
          top = fmaxf(top, fmaxf(fabsf(t.x), fabsf(t.y)));
        }
      }
    } else {
#pragma unroll
      for (int w = 0; w < G; ++w)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[w][j] = 0.f;
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    int e = static_cast<int>(__float_as_uint(top) >> 23) - 127 - 10;
    e = max(min(e, 100), -100);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);   // 2^-e
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
    for (int w = 0; w < G; ++w) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[w][j] *= down;
        sum += x[w][j];
      }
      f.frag[nt][w][0] = from_f32x2<false>(x[w][0], x[w][4]);
      f.frag[nt][w][1] = from_f32x2<false>(x[w][2], x[w][6]);
      // their codes stand four bits higher
      f.frag[nt][w][2] = from_f32x2<false>(x[w][1] * 0.0625f, x[w][5] * 0.0625f);
      f.frag[nt][w][3] = from_f32x2<false>(x[w][3] * 0.0625f, x[w][7] * 0.0625f);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= 5.9604644775390625e-8f;   // 2^-24
      f.sums[nt][w][0] = __shfl_sync(0xffffffffu, sum, 8 * q4);
      f.sums[nt][w][1] = __shfl_sync(0xffffffffu, sum, 8 * q4 + 4);
    }
    const float factor = up * 16777216.f * (a.sm_scale * kLog2e);
    f.factor[nt][0] = __shfl_sync(0xffffffffu, factor, 8 * q4);
    f.factor[nt][1] = __shfl_sync(0xffffffffu, factor, 8 * q4 + 4);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = row0 + 8 * nt + 2 * q4 + j, i = r / rows.group;
      f.last[nt][j] = r < rows.count && i < count ? n - count + i : -1;
    }
  }
}

// ------------------------------------------------------------------ one block of 16 tokens
// Scores of tokens (g, g + 8) (g = lane / 4) and query rows (2 c, 2 c + 1) from the records at `rec`, in log2 units.
template <int D, int NT, bool kBf16>
__device__ __forceinline__ void block_scores(float (&s)[NT][4], const uint8_t* rec, const Query<D, NT>& f) {
  using R = Record<D>;
  constexpr int G = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const uint8_t* lo = rec + g * R::kBytes;
  const uint8_t* hi = lo + 8 * R::kBytes;
  uint32_t kl[G], kh[G], pl[G], ph[G];
  if constexpr (G == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(lo + 8 * q4), v = *reinterpret_cast<const uint2*>(hi + 8 * q4);
    kl[0] = u.x, kl[1] = u.y, kh[0] = v.x, kh[1] = v.y;
    const uint2 x = *reinterpret_cast<const uint2*>(lo + R::kKPairs), y = *reinterpret_cast<const uint2*>(hi + R::kKPairs);
    pl[0] = x.x, pl[1] = x.y, ph[0] = y.x, ph[1] = y.y;
  } else {
#pragma unroll
    for (int q = 0; q < G / 4; ++q) {
      const uint4 u = *reinterpret_cast<const uint4*>(lo + 64 * q + 16 * q4), v = *reinterpret_cast<const uint4*>(hi + 64 * q + 16 * q4);
      kl[4 * q] = u.x, kl[4 * q + 1] = u.y, kl[4 * q + 2] = u.z, kl[4 * q + 3] = u.w;
      kh[4 * q] = v.x, kh[4 * q + 1] = v.y, kh[4 * q + 2] = v.z, kh[4 * q + 3] = v.w;
      const uint4 x = *reinterpret_cast<const uint4*>(lo + R::kKPairs + 16 * q), y = *reinterpret_cast<const uint4*>(hi + R::kKPairs + 16 * q);
      pl[4 * q] = x.x, pl[4 * q + 1] = x.y, pl[4 * q + 2] = x.z, pl[4 * q + 3] = x.w;
      ph[4 * q] = y.x, ph[4 * q + 1] = y.y, ph[4 * q + 2] = y.z, ph[4 * q + 3] = y.w;
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[nt][j] = 0.f;
#pragma unroll
  for (int w = 0; w < G; ++w) {
    const uint32_t a8 = kl[w] >> 8, b8 = kh[w] >> 8;
    const float2 sl = to_f32x2<kBf16>(pl[w]), sh = to_f32x2<kBf16>(ph[w]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float acc[4];
      mma_f16_first(acc, kl[w] & 0x000f000fu, kh[w] & 0x000f000fu, a8 & 0x000f000fu, b8 & 0x000f000fu, f.frag[nt][w][0], f.frag[nt][w][1]);
      mma_f16(acc, kl[w] & 0x00f000f0u, kh[w] & 0x00f000f0u, a8 & 0x00f000f0u, b8 & 0x00f000f0u, f.frag[nt][w][2], f.frag[nt][w][3]);
      s[nt][0] = fmaf(sl.x, acc[0], fmaf(sl.y, f.sums[nt][w][0], s[nt][0]));
      s[nt][1] = fmaf(sl.x, acc[1], fmaf(sl.y, f.sums[nt][w][1], s[nt][1]));
      s[nt][2] = fmaf(sh.x, acc[2], fmaf(sh.y, f.sums[nt][w][0], s[nt][2]));
      s[nt][3] = fmaf(sh.x, acc[3], fmaf(sh.y, f.sums[nt][w][1], s[nt][3]));
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[nt][j] *= f.factor[nt][j & 1];
}

// The sums of one piece of an item.
template <int D, int NT>
struct Sums {
  static constexpr int G = D / 32;
  float o[2 * G][NT][4];       // tile 2 w + t: dims 32 w + 4 g + 2 t (times 2^-24) and + 1 (times 2^-20), both over `unit`
  float minima[G][NT][2];      // this lane's share of sum p m, rows 2 c, 2 c + 1
  float l[NT][2], ref[NT][2];
  float unit;                  // power of two that p * s is divided by
};

template <int D, int NT>
__device__ __forceinline__ void clear(Sums<D, NT>& x) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < 2 * (D / 32); ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) x.o[j][nt][i] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int w = 0; w < D / 32; ++w) x.minima[w][nt][i] = 0.f;
      x.l[nt][i] = 0.f;
      x.ref[nt][i] = -INFINITY;
    }
  }
  x.unit = 1.17549435e-38f;
}

// The second product of 16 tokens: p of tokens (g, g + 8), zero where hidden; `left`: tokens of the block that exist.
template <int D, int NT, bool kBf16>
__device__ __forceinline__ void block_output(Sums<D, NT>& x, const float (&p)[NT][4], const uint8_t* rec, const float2 (&lo_pair)[D / 32],
                                             const float2 (&hi_pair)[D / 32], float per_unit) {
  using R = Record<D>;
  constexpr int G = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  constexpr int kWords = G / 2;                  // 32-bit words of one token's V codes in a lane
  uint32_t v[4][kWords];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint8_t* at = rec + (2 * q4 + (j & 1) + 8 * (j >> 1)) * R::kBytes + R::kVCodes + g * (D / 16);
    if constexpr (kWords == 1) {
      v[j][0] = *reinterpret_cast<const uint32_t*>(at);
    } else if constexpr (kWords == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(at);
      v[j][0] = u.x, v[j][1] = u.y;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(at);
      v[j][0] = u.x, v[j][1] = u.y, v[j][2] = u.z, v[j][3] = u.w;
    }
  }
#pragma unroll
  for (int w = 0; w < G; ++w) {
    // the half words of group w: low half token 2 c (2 c + 8), high half the token behind it
    const uint32_t pick = (w & 1) ? 0x7632u : 0x5410u;
    const uint32_t y = __byte_perm(v[0][w / 2], v[1][w / 2], pick), z = __byte_perm(v[2][w / 2], v[3][w / 2], pick);
    const uint32_t y8 = y >> 8, z8 = z >> 8;
    const float sl = lo_pair[w].x * per_unit, sh = hi_pair[w].x * per_unit;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t b0 = transpose_8x8(from_f32x2<false>(p[nt][0] * sl, p[nt][1] * sl));
      const uint32_t b1 = transpose_8x8(from_f32x2<false>(p[nt][2] * sh, p[nt][3] * sh));
      mma_f16(x.o[2 * w][nt], y & 0x000f000fu, y & 0x00f000f0u, z & 0x000f000fu, z & 0x00f000f0u, b0, b1);
      mma_f16(x.o[2 * w + 1][nt], y8 & 0x000f000fu, y8 & 0x00f000f0u, z8 & 0x000f000fu, z8 & 0x00f000f0u, b0, b1);
      x.minima[w][nt][0] = fmaf(p[nt][0], lo_pair[w].y, fmaf(p[nt][2], hi_pair[w].y, x.minima[w][nt][0]));
      x.minima[w][nt][1] = fmaf(p[nt][1], lo_pair[w].y, fmaf(p[nt][3], hi_pair[w].y, x.minima[w][nt][1]));
    }
  }
}

// Scales and minima of V of tokens (g, g + 8); zero for tokens that do not exist (what the page holds there may be NaN).
template <int D, bool kBf16>
__device__ __forceinline__ void value_pairs(float2 (&lo)[D / 32], float2 (&hi)[D / 32], const uint8_t* rec, int left) {
  using R = Record<D>;
  const int g = (threadIdx.x & 31) >> 2;
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    const uint32_t a = g < left ? *reinterpret_cast<const uint32_t*>(rec + g * R::kBytes + R::kVPairs + 4 * w) : 0u;
    const uint32_t b = g + 8 < left ? *reinterpret_cast<const uint32_t*>(rec + (g + 8) * R::kBytes + R::kVPairs + 4 * w) : 0u;
    lo[w] = to_f32x2<kBf16>(a);
    hi[w] = to_f32x2<kBf16>(b);
  }
}

// One tile of 32 tokens: `rec` the records of its two blocks (null: the page is not there), `left` its tokens.
template <int D, int NT, bool kBf16>
__device__ __forceinline__ void one_tile(Sums<D, NT>& x, const Query<D, NT>& f, const uint8_t* const (&rec)[2], int slot, int left) {
  constexpr int G = D / 32;
  const int g = (threadIdx.x & 31) >> 2;
  float s[2][NT][4];
  float top[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (16 * k < left && rec[k] != nullptr) {
      block_scores<D, NT, kBf16>(s[k], rec[k], f);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (slot + 16 * k + g + 8 * (j >> 1) > f.last[nt][j & 1]) s[k][nt][j] = -INFINITY;
          top[nt][j & 1] = fmaxf(top[nt][j & 1], s[k][nt][j]);
        }
    }
  }
  bool raise = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) raise |= top[nt][0] > x.ref[nt][0] + kRaise || top[nt][1] > x.ref[nt][1] + kRaise;
  if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float m = top[nt][i];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const float ref = fmaxf(m, x.ref[nt][i]);
        const float by = ref == -INFINITY ? 1.f : ex2(x.ref[nt][i] - ref);
        x.ref[nt][i] = ref;
        x.l[nt][i] *= by;
#pragma unroll
        for (int w = 0; w < G; ++w) x.minima[w][nt][i] *= by;
#pragma unroll
        for (int j = 0; j < 2 * G; ++j) {
          x.o[j][nt][i] *= by;
          x.o[j][nt][i + 2] *= by;
        }
      }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (16 * k < left && rec[k] != nullptr) {
      float2 lo[G], hi[G];
      value_pairs<D, kBf16>(lo, hi, rec[k], left - 16 * k);
      float widest = 0.f;
#pragma unroll
      for (int w = 0; w < G; ++w) widest = fmaxf(widest, fmaxf(lo[w].x, hi[w].x));
      if (__any_sync(0xffffffffu, widest > x.unit * kRaiseScale)) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) widest = fmaxf(widest, __shfl_xor_sync(0xffffffffu, widest, d));
        // the power of two below it, and no less than can be divided by
        const float unit = fmaxf(__uint_as_float(__float_as_uint(widest) & 0x7f800000u), 1.17549435e-38f);
        const float by = x.unit / unit;
#pragma unroll
        for (int j = 0; j < 2 * G; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) x.o[j][nt][i] *= by;
        x.unit = unit;
      }
      float p[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // a row that sees nothing yet has no reference to subtract
          p[nt][j] = s[k][nt][j] == -INFINITY ? 0.f : ex2(s[k][nt][j] - x.ref[nt][j & 1]);
          x.l[nt][j & 1] += p[nt][j];
        }
      block_output<D, NT, kBf16>(x, p, rec[k], lo, hi, 1.f / x.unit);
    }
  }
}

// ------------------------------------------------------------------ results
// Piece `slot` (0: a share's first item, 1: its last) of a worker: per query row D sums, the reference and the sum
// of the weights.
template <int D, int NT>
__host__ __device__ constexpr int piece_floats() { return 8 * NT * (D + 2); }

template <int D, int NT, bool kBf16>
__device__ __forceinline__ void store_sums(Sums<D, NT>& x, const Cache4Attention& a, const Rows& rows, int b, int h, int row0, float* piece) {
  constexpr int G = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  // codes back from their places in a word, then what p * s was divided by
  auto low = [&](float v) { return v * 16777216.f * x.unit; };
  auto high = [&](float v) { return v * 1048576.f * x.unit; };
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        x.l[nt][i] += __shfl_xor_sync(0xffffffffu, x.l[nt][i], d);
#pragma unroll
        for (int w = 0; w < G; ++w) x.minima[w][nt][i] += __shfl_xor_sync(0xffffffffu, x.minima[w][nt][i], d);
      }
      const int r = 8 * nt + 2 * q4 + i, row = row0 + r;
      if (row >= rows.count) continue;
      const float l = x.l[nt][i];
      if (piece != nullptr) {
        float* dst = piece + r * (D + 2);
#pragma unroll
        for (int w = 0; w < G; ++w) {
          const float m = x.minima[w][nt][i];
          *reinterpret_cast<float2*>(dst + 32 * w + 4 * g) = make_float2(low(x.o[2 * w][nt][i]) + m, high(x.o[2 * w][nt][i + 2]) + m);
          *reinterpret_cast<float2*>(dst + 32 * w + 4 * g + 2) = make_float2(low(x.o[2 * w + 1][nt][i]) + m, high(x.o[2 * w + 1][nt][i + 2]) + m);
        }
        if (g == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(x.ref[nt][i], l);
      } else {
        const int t = row / rows.group, hq = h * rows.group + row - t * rows.group;
        const float inv = l == 0.f ? 0.f : 1.f / l;      // a row that sees nothing is zero
        uint16_t* dst = static_cast<uint16_t*>(a.o) + b * a.o_stride[0] + hq * a.o_stride[1] + t * a.o_stride[2];
#pragma unroll
        for (int w = 0; w < G; ++w) {
          const float m = x.minima[w][nt][i];
          const uint2 v = make_uint2(from_f32x2<kBf16>((low(x.o[2 * w][nt][i]) + m) * inv, (high(x.o[2 * w][nt][i + 2]) + m) * inv),
                                     from_f32x2<kBf16>((low(x.o[2 * w + 1][nt][i]) + m) * inv, (high(x.o[2 * w + 1][nt][i + 2]) + m) * inv));
          *reinterpret_cast<uint2*>(dst + 32 * w + 4 * g) = v;
        }
        if (g == 0 && a.lse != nullptr)
          a.lse[(static_cast<int64_t>(b) * a.Hq + hq) * a.S + t] = l == 0.f ? -INFINITY : (x.ref[nt][i] + __log2f(l)) * kLn2;
      }
    }
  }
}

// A place in the list of tiles: item `item` of sequence b, tile t of `tiles`.
struct Cursor {
  int b, n, tiles, item, t;
  long long left;          // tiles of the share from here on
};
__device__ __forceinline__ Cursor cursor_at(const Cache4& c, const int* counts, int per_sequence, long long at, long long end) {
  Cursor k;
  long long first;
  k.b = sequence_of(c, counts, per_sequence, at, &first, &k.tiles);
  k.n = tokens_of(c, k.b);
  k.item = static_cast<int>((at - first) / k.tiles);
  k.t = static_cast<int>(at - first - static_cast<long long>(k.item) * k.tiles);
  k.left = end - at;
  return k;
}
__device__ __forceinline__ void advance(Cursor& k, const Cache4& c, const int* counts, int per_sequence) {
  --k.left;
  if (++k.t < k.tiles || k.left == 0) return;
  k.t = 0;
  if (++k.item < per_sequence) return;
  k.item = 0;
  do {                     // the next sequence that has tokens: there is one, tiles are left
    k.tiles = tiles_of(c, counts, ++k.b);
  } while (k.tiles == 0);
  k.n = tokens_of(c, k.b);
}

// Every warp works for itself: a ring of tiles in shared memory, which its first lane fills with bulk copies as soon
// as the warp is done with a slot, across the items of its share.
template <int D, int NT, bool kBf16>
__global__ void __launch_bounds__(kThreads, (Shape<D, NT>::kCtas)) cache4_attention_kernel(const Cache4 c, const Cache4Attention a, const Rows rows,
                                                                                        const int row_blocks, const unsigned long long wait_limit_ns) {
  using R = Record<D>;
  using Sh = Shape<D, NT>;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t full_bar[kWarps * Sh::kStages];
  __shared__ int abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < kWarps * Sh::kStages) mbar_init(smem_u32(&full_bar[threadIdx.x]), 1);
  if (threadIdx.x == 0) abort_word = 0;
  fence_barrier_init();
  fence_proxy_async();
  __syncthreads();
  griddep_launch_dependents();
  griddep_wait();
  const int per_sequence = c.H * row_blocks;
  const long long total = tiles_before(c, a.counts, c.B) * per_sequence;
  const long long worker = worker_here(), workers = workers_used(total, static_cast<long long>(gridDim.x) * kWarps);
  if (worker >= workers) return;
  Cursor use = cursor_at(c, a.counts, per_sequence, share_begin(total, worker, workers), share_begin(total, worker + 1, workers));
  Cursor load = use;
  const uint8_t* const my_ring = ring + warp * Sh::kStages * Sh::kSlotBytes;
  const uint32_t my_bar = smem_u32(&full_bar[warp * Sh::kStages]);
  const int mask = (1 << c.page_shift) - 1;
  const bool split = c.page_shift == 4;    // a tile is two pages

  // Pages of tiles window .. window + 31 of sequence window_b, one per lane (two where a tile is two pages).
  int window_b = -1, window = 0, page_lo = 0, page_hi = 0;
  uint32_t have = 0;                       // two bits per slot: which halves of its tile are there
  auto issue = [&](int stage) {
    if (load.b != window_b || load.t < window || load.t >= window + 32) {
      window_b = load.b;
      window = load.t;
      const int slot = (window + lane) * kTile;
      const int* row = c.table + static_cast<int64_t>(load.b) * c.table_stride;
      page_lo = slot < load.n ? row[slot >> c.page_shift] : 0;
      page_hi = split && slot + 16 < load.n ? row[(slot + 16) >> 4] : 0;
    }
    const int lo = __shfl_sync(0xffffffffu, page_lo, load.t - window), hi = __shfl_sync(0xffffffffu, page_hi, load.t - window);
    const int slot = load.t * kTile, left = load.n - slot;
    const bool lo_ok = static_cast<unsigned>(lo) < static_cast<unsigned>(c.pages);
    const bool hi_there = left > 16, hi_ok = split ? static_cast<unsigned>(hi) < static_cast<unsigned>(c.pages) : lo_ok;
    if (!(lo_ok && (hi_ok || !hi_there))) report_bad_index(c.status, kTagCachePage);
    have = (have & ~(3u << (2 * stage))) | ((lo_ok ? 1u : 0u) | (hi_there && hi_ok ? 2u : 0u)) << (2 * stage);
    if (lane == 0) {
      constexpr uint32_t kHalf = 16 * R::kBytes;
      const uint32_t bar = my_bar + 8 * stage, dst = smem_u32(my_ring + stage * Sh::kSlotBytes);
      const int h = load.item / row_blocks;
      const uint8_t* head = c.kv + h * c.kv_stride[1] + static_cast<int64_t>(slot & mask) * R::kBytes;
      if (split) {
        mbar_arrive_expect_tx(bar, (lo_ok ? kHalf : 0u) + (hi_there && hi_ok ? kHalf : 0u));
        if (lo_ok) bulk_load(dst, head + lo * c.kv_stride[0], bar, kHalf);
        if (hi_there && hi_ok) bulk_load(dst + kHalf, head + hi * c.kv_stride[0], bar, kHalf);
      } else {
        const uint32_t bytes = !lo_ok ? 0u : hi_there ? 2 * kHalf : kHalf;
        mbar_arrive_expect_tx(bar, bytes);
        if (lo_ok) bulk_load(dst, head + lo * c.kv_stride[0], bar, bytes);
      }
    }
    advance(load, c, a.counts, per_sequence);
  };
#pragma unroll 1
  for (int i = 0; i < Sh::kStages && load.left > 0; ++i) issue(i);

  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  while (use.left > 0) {
    // one piece: the tiles of one item that belong to this share
    const int b = use.b, t0 = use.t, tiles = use.tiles, h = use.item / row_blocks, row0 = (use.item - h * row_blocks) * 8 * NT, n = use.n;
    const int t1 = static_cast<int>(min(static_cast<long long>(tiles), t0 + use.left));
    Query<D, NT> f;
    load_query<D, NT, kBf16>(f, c, a, rows, b, h, row0, n);
    Sums<D, NT> x;
    clear(x);
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      ok = ok && mbar_wait_warp(my_bar + 8 * stage, phase, &abort_word, wait_limit_ns, kTagCache4Load);
      if (!ok) break;
      const uint8_t* slot = my_ring + stage * Sh::kSlotBytes;
      const uint8_t* rec[2] = {(have >> (2 * stage)) & 1 ? slot : nullptr, (have >> (2 * stage)) & 2 ? slot + 16 * R::kBytes : nullptr};
      one_tile<D, NT, kBf16>(x, f, rec, t * kTile, n - t * kTile);
      __syncwarp();
      if (load.left > 0) issue(stage);
      if (++stage == Sh::kStages) {
        stage = 0;
        phase ^= 1;
      }
      advance(use, c, a.counts, per_sequence);
    }
    if (!ok) break;
    float* piece = nullptr;
    if (t0 > 0 || t1 < tiles) piece = a.pieces + (worker * 2 + (t0 == 0)) * piece_floats<D, NT>();
    store_sums<D, NT, kBf16>(x, a, rows, b, h, row0, piece);
  }
  if (!ok) {
    // a copy did not arrive in time: said in the status word; no copy is left behind without a second wait
    if (lane == 0) atomicCAS(c.status, 0, abort_word);
    for (int i = 0; i < Sh::kStages; ++i) {
      int again = 0;
      mbar_wait(my_bar + 8 * i, i < stage ? phase ^ 1 : phase, &again, wait_limit_ns, kTagCache4Load);
    }
  }
}

// One CTA per query row of an item: joins the item's pieces where there are several, and answers for items without
// tokens.  The order of the pieces is that of the tokens, so results do not depend on timing.
template <int D, int NT, bool kBf16>
__global__ void __launch_bounds__(kJoinThreads) cache4_join_kernel(const Cache4 c, const Cache4Attention a, const Rows rows, const int row_blocks,
                                                                   const long long all_workers) {
  constexpr int kJoinWarps = kJoinThreads / 32;
  constexpr int kEach = D / 32;
  __shared__ float part[kJoinWarps][D];
  griddep_launch_dependents();
  griddep_wait();
  const int row = blockIdx.x % rows.count;
  const int bh = blockIdx.x / rows.count, b = bh / c.H, h = bh - b * c.H;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = tiles_of(c, a.counts, b);
  const int t = row / rows.group, hq = h * rows.group + row - t * rows.group;
  uint16_t* dst = static_cast<uint16_t*>(a.o) + b * a.o_stride[0] + hq * a.o_stride[1] + t * a.o_stride[2];
  float* lse = a.lse != nullptr ? a.lse + (static_cast<int64_t>(b) * a.Hq + hq) * a.S + t : nullptr;
  if (tiles == 0) {
    for (int d = threadIdx.x; d < D; d += kJoinThreads) dst[d] = 0;
    if (threadIdx.x == 0 && lse != nullptr) *lse = -INFINITY;
    return;
  }
  const int per_sequence = c.H * row_blocks;
  const long long total = tiles_before(c, a.counts, c.B) * per_sequence;
  const long long workers = workers_used(total, all_workers);
  const int block = row / (8 * NT), r = row - block * 8 * NT;
  const long long first = tiles_before(c, a.counts, b) * per_sequence + static_cast<long long>(h * row_blocks + block) * tiles;
  const long long w0 = worker_of(total, first, workers), w1 = worker_of(total, first + tiles - 1, workers);
  if (w0 == w1) return;                       // in one piece: answered already
  const int pieces = static_cast<int>(w1 - w0) + 1;
  auto piece_of = [&](int i) {                // the first one is its worker's last item, the others their workers' first
    return a.pieces + ((w0 + i) * 2 + (i == 0)) * piece_floats<D, NT>() + r * (D + 2);
  };
  float ref = -INFINITY;
  for (int i = lane; i < pieces; i += 32) ref = fmaxf(ref, piece_of(i)[D]);
#pragma unroll
  for (int d = 16; d; d >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, d));
  float l = 0.f;
  for (int i = lane; i < pieces; i += 32) {
    const float* p = piece_of(i);
    // what a piece that saw nothing holds: no reference and a sum of zero
    l += p[D] == -INFINITY ? p[D + 1] : ex2(p[D] - ref) * p[D + 1];
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  float sum[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) sum[j] = 0.f;
#pragma unroll 4
  for (int i = warp; i < pieces; i += kJoinWarps) {
    const float* p = piece_of(i);
    const float by = p[D] == -INFINITY ? 1.f : ex2(p[D] - ref);
#pragma unroll
    for (int j = 0; j < kEach; ++j) sum[j] += by * p[lane + 32 * j];
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j) part[warp][lane + 32 * j] = sum[j];
  __syncthreads();
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int d = threadIdx.x; d < D; d += kJoinThreads) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) o += part[w][d];
    dst[d] = from_f32<kBf16>(o * inv);
  }
  if (threadIdx.x == 0 && lse != nullptr) *lse = l == 0.f ? -INFINITY : (ref + __log2f(l)) * kLn2;
}

// The weights: every token's softmax weights over all query rows of its K/V head, added to weight[].  The scores are
// computed again from K, against the rows' log-sum-exp; a token belongs to one warp, so nothing is added twice at once.
template <int D, int NT, bool kBf16>
__global__ void __launch_bounds__(kThreads) cache4_weight_kernel(const Cache4 c, const Cache4Attention a, const Rows rows, const int row_blocks) {
  using R = Record<D>;
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const long long total = tiles_before(c, a.counts, c.B) * c.H;
  const long long worker = worker_here(), workers = workers_used(total, static_cast<long long>(gridDim.x) * kWarps);
  if (worker >= workers) return;
  long long at = share_begin(total, worker, workers);
  const long long end = share_begin(total, worker + 1, workers);
  long long first;
  int tiles;
  int b = sequence_of(c, a.counts, c.H, at, &first, &tiles);
  const int mask = (1 << c.page_shift) - 1;
  while (at < end) {
    if (at >= first + static_cast<long long>(tiles) * c.H) b = sequence_of(c, a.counts, c.H, at, &first, &tiles);
    const int h = static_cast<int>((at - first) / tiles);
    const int t0 = static_cast<int>(at - first - static_cast<long long>(h) * tiles);
    const int t1 = static_cast<int>(min(static_cast<long long>(tiles), t0 + end - at));
    const int n = tokens_of(c, b);
    for (int block = 0; block < row_blocks; ++block) {
      Query<D, NT> f;
      load_query<D, NT, kBf16>(f, c, a, rows, b, h, 8 * NT * block, n);
      float lse[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = 8 * (NT * block + nt) + 2 * q4 + i, t = row / rows.group, hq = h * rows.group + row - t * rows.group;
          lse[nt][i] = f.last[nt][i] >= 0 ? a.lse[(static_cast<int64_t>(b) * a.Hq + hq) * a.S + t] * kLog2e : 0.f;
        }
      for (int t = 2 * t0; t < 2 * t1; ++t) {
        const int slot = 16 * t;
        int64_t page;
        if (slot >= n || !find_page(c, b, slot, &page)) continue;
        float s[NT][4];
        block_scores<D, NT, kBf16>(s, c.kv + page * c.kv_stride[0] + h * c.kv_stride[1] + static_cast<int64_t>(slot & mask) * R::kBytes, f);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (slot + g + 8 * (j >> 1) <= f.last[nt][j & 1]) sum[j >> 1] += ex2(s[nt][j] - lse[nt][j & 1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
          sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
          if (q4 == 0 && slot + g + 8 * i < n)
            c.weight[page * c.weight_stride[0] + h * c.weight_stride[1] + (slot & mask) + g + 8 * i] += sum[i];
        }
      }
    }
    at += t1 - t0;
  }
}

template <int D, int NT, bool kBf16>
cudaError_t launch_one(const Cache4& c, const Cache4Attention& a, int sm_count, cudaStream_t stream, long long* launches) {
  Rows rows;
  rows.group = a.Hq / c.H;
  rows.count = rows.group * a.S;
  const int row_blocks = (rows.count + 8 * NT - 1) / (8 * NT);
  using Sh = Shape<D, NT>;
  const int grid = sm_count * Sh::kCtas;
  const bool pdl = option_pdl() != 0;
  static std::atomic<unsigned long long> smem_done{0};   // per kernel instantiation, bit per device
  cudaError_t e = set_dynamic_smem_once(smem_done, reinterpret_cast<const void*>(cache4_attention_kernel<D, NT, kBf16>), Sh::kRingBytes);
  if (e != cudaSuccess) return e;
  e = launch_persistent(cache4_attention_kernel<D, NT, kBf16>, grid, kThreads, Sh::kRingBytes, stream, pdl, c, a, rows, row_blocks, option_wait_limit_ns());
  if (e != cudaSuccess) return e;
  *launches += 1;
  e = launch_persistent(cache4_join_kernel<D, NT, kBf16>, c.B * c.H * rows.count, kJoinThreads, 0, stream, pdl, c, a, rows, row_blocks,
                        static_cast<long long>(grid) * kWarps);
  if (e != cudaSuccess) return e;
  *launches += 1;
  if (c.weight != nullptr) {
    e = launch_persistent(cache4_weight_kernel<D, NT, kBf16>, 2 * sm_count, kThreads, 0, stream, pdl, c, a, rows, row_blocks);
    if (e == cudaSuccess) *launches += 1;
  }
  return e;
}

// Sixteen query rows at a time where there are more than eight: the cache is read half as often.  At D = 256 the
// accumulators of sixteen rows leave no room for anything else.
bool sixteen_rows(int D, int rows) { return D <= 128 && rows > 8; }

template <int D>
cudaError_t launch_dim(const Cache4& c, const Cache4Attention& a, int sm_count, cudaStream_t stream, long long* launches) {
  if constexpr (D <= 128) {
    if (sixteen_rows(D, a.Hq / c.H * a.S))
      return c.bf16 ? launch_one<D, 2, true>(c, a, sm_count, stream, launches) : launch_one<D, 2, false>(c, a, sm_count, stream, launches);
  }
  return c.bf16 ? launch_one<D, 1, true>(c, a, sm_count, stream, launches) : launch_one<D, 1, false>(c, a, sm_count, stream, launches);
}

}  // namespace

template <int D, int NT>
size_t pieces_bytes(int sm_count) {
  return static_cast<size_t>(sm_count) * Shape<D, NT>::kCtas * kWarps * 2 * piece_floats<D, NT>() * sizeof(float);
}
size_t cache4_attention_workspace(int D, int Hq, int H, int S, int sm_count) {
  const bool wide = sixteen_rows(D, Hq / H * S);
  if (D == 64) return wide ? pieces_bytes<64, 2>(sm_count) : pieces_bytes<64, 1>(sm_count);
  if (D == 128) return wide ? pieces_bytes<128, 2>(sm_count) : pieces_bytes<128, 1>(sm_count);
  return pieces_bytes<256, 1>(sm_count);
}

cudaError_t launch_cache4_attention(const Cache4& c, const Cache4Attention& a, int sm_count, cudaStream_t stream, long long* launches) {
  switch (c.D) {
    case 64: return launch_dim<64>(c, a, sm_count, stream, launches);
    case 128: return launch_dim<128>(c, a, sm_count, stream, launches);
    case 256: return launch_dim<256>(c, a, sm_count, stream, launches);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace rsfa
