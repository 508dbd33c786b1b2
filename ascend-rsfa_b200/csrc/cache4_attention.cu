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
// The second product runs over codes less their middle, u - 8 (exact), and the middles m + 8 s of the groups are a third,
// small one: what rounding p * s to fp16 leaves is then in proportion to a group's range.  p itself is 32 bits wide where
// it is summed and added to the weights; the middles take it as two numbers of the cache's type.
//
// Rows of scores are handed on by a flash recurrence whose reference is raised only when a score exceeds what it
// was set for by a log2 unit.
//
// The work is the list of all tiles of 32 (64) tokens of all (sequence, K/V head, block of query rows), and every warp of
// the device takes an equal, contiguous share of it, whatever the lengths are.  A share's first and last item may
// continue in other warps: their sums go to a workspace and a second kernel joins them.
//
// What bounds it: not HBM, 5 D / 4 bytes per token and K/V head, but some 355 instructions per 16 tokens, K/V head and 8
// rows (528 for 16), at the rate at which three warps per scheduler (two), all that registers allow, keep it busy: 57 % of the
// issue slots (49 %).
// (Tensor cores of the newer kind want 128-row operands in shared memory; here 8 rows meet codes that exist unpacked in
// registers only.)  Times with 128 dims, against the time for the bytes alone: one sequence of 131072 tokens,
// 8 heads, 51.2 us (25.6; 3.3 TB/s); 64 sequences of 1 to 8192 tokens, 32 heads over 8, 87 us (53); 256 sequences of 200
// tokens 40.6 us (11); one of 500 tokens 9.5 us, two dependent kernels.
//
// More than 16 rows are blocks of 16 (8 at D = 256) that each read and unpack the cache again: made for decoding and a few tokens to
// verify.  512 new tokens over 8192 held, 32 heads over 8 of 128 dims, take 491 us (144 TFLOP/s, 9 % of the dense rate), 2048 2.2 ms.
#include "../../include/rsfa.h"
#include "ops_common.cuh"

namespace rsfa {
namespace {

constexpr int kWeightWarps = 4, kWeightThreads = 32 * kWeightWarps;
constexpr int kJoinThreads = 128, kJoinMost = 512;
// Tokens per tile: what a tile costs apart from its tokens is spread over 5 KB (10 KB) of them.
__host__ __device__ constexpr int tile_tokens(int D) { return D == 64 ? 64 : 32; }
// One CTA per multiprocessor: as many warps as the registers of their accumulators allow, and slots of a warp's ring by the
// shared memory that is left.  (When they were measured: three CTAs of four warps, the same loop, but three times the CTAs to
// start, 256 sequences of 200 tokens in 48 us for 39.  Sixteen rows of 64 dims by 8 warps without spills, 16 sequences of 16384
// tokens, 64 heads over 4, in 45.3 us; by 12 with them in 49.2.  Eight rows by 16 warps with two slots: 32 sequences of 16384
// tokens 85.7 us for 89.3, 16 of up to 2048 tokens 24.1 for 21.5, left at 12.)
template <int D, int NT>
struct Shape {
  static constexpr int kWarps = D == 256 || NT == 2 ? 8 : 12, kThreads = 32 * kWarps;
  static constexpr int kStages = D == 256 ? 2 : NT == 2 ? 4 : 3;
  static constexpr int kTile = tile_tokens(D);
  static constexpr int kPieces = kTile / 16;     // loads per tile: a page holds whole ones
  static constexpr int kPieceBytes = 16 * Record<D>::kBytes;
  static constexpr int kSlotBytes = kTile * Record<D>::kBytes;
  static constexpr int kRingBytes = kWarps * kStages * kSlotBytes;
};
constexpr int kItemCost = 2;         // tiles that an item takes as long as beside its own, see all_units
constexpr int kTagCache4Load = 40;   // of a bounded wait, in the status word
// A reference is set kHeadroom log2 units below its row's largest score and raised when a score is kRaise above it, one unit
// above the largest before; the scales' unit is raised when one is kRaiseScale of it.  So a product p * s is at most 2^11 * 4
// in fp16, whose normal numbers then reach weights of 2^-24 of the largest, and the largest weights, which are what rounding
// shows in most, are close to powers of two (fp16, whose own rounding is 2.1e-4: 4 sequences of up to 8192 tokens, 64 of 1 to 8192 and
// one of 60000, results off by 2.4e-4, 2.6e-4 and 2.5e-4; raised only eight units above, the first and the last: 2.8e-4 and 3.5e-4).
constexpr float kHeadroom = 10.f, kRaise = 11.f;
constexpr float kRaiseScale = 4.f;
constexpr float kFar = 256.f;        // see raise()

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(b0));
}
// The 16-bit numbers of the cache's own type.
template <bool kBf16>
__device__ __forceinline__ void mma_own_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  if constexpr (kBf16)
    asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(b0));
  else
    mma_f16_k8(c, a0, a1, b0);
}
template <bool kBf16>
__device__ __forceinline__ void mma_own(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    mma_f16(c, a0, a1, a2, a3, b0, b1);
}
// Pairs of codes as (u - 8) * 2^-9: as the numbers u * 2^-24 that they are (kUp: u * 2^-20, four bits further up).
template <bool kUp>
__device__ __forceinline__ uint32_t centred(uint32_t codes) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(codes), "r"(kUp ? 0x68006800u : 0x78007800u), "r"(0xa400a400u));
  return r;
}
// The low half of a pair, a number of the cache's type, times another such number: conversion and factor in one.
template <bool kBf16>
__device__ __forceinline__ float scale_of(uint32_t pair, uint16_t by) {
  float r;
  if constexpr (kBf16)
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\nfma.rn.f32.bf16 %0, l, %2, %3;\n}\n" : "=f"(r) : "r"(pair), "h"(by), "f"(0.f));
  else
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\nfma.rn.f32.f16 %0, l, %2, %3;\n}\n" : "=f"(r) : "r"(pair), "h"(by), "f"(0.f));
  return r;
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

// The kernels behind the attention kernel read lengths and counts ahead of their wait for it.  What wrote these is complete, the
// attention kernel has waited for it; the fence is there so that this multiprocessor's L1 has no older copy of them.
__device__ __forceinline__ void fence_ahead() { __threadfence(); }

// ------------------------------------------------------------------ the list of tiles
// Items are (sequence, K/V head, block of query rows) in this order, an item's tiles follow one another.
__device__ __forceinline__ int visible_tokens(const Cache4& c, const int* counts, int b) {
  return counts != nullptr && counts[b] <= 0 ? 0 : tokens_of(c, b);
}
__device__ __forceinline__ int tiles_of(const Cache4& c, const int* counts, int b) {
  const int shift = c.D == 64 ? 6 : 5;
  return (visible_tokens(c, counts, b) + (1 << shift) - 1) >> shift;
}
// What is divided among the warps: an item of n tiles is n + cost units, cost of them in front for what an item takes by
// itself (its query rows, its results).  Short items would otherwise make the shares that have many of them the last
// ones: 64 sequences of 1 to 8192 tokens 103 -> 86 us when it was measured (94 with a cost of one tile, 85 and 86 with three and four).
//
// One warp: units of all sequences and of those before b, per K/V head and block of rows.
__device__ __forceinline__ long long all_units(const Cache4& c, const int* counts, int cost, int b, long long* before) {
  long long n = 0, m = 0;
  for (int i = threadIdx.x & 31; i < c.B; i += 32) {
    const int tiles = tiles_of(c, counts, i), units = tiles > 0 ? tiles + cost : 0;
    n += units;
    m += i < b ? units : 0;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    n += __shfl_xor_sync(0xffffffffu, n, d);
    m += __shfl_xor_sync(0xffffffffu, m, d);
  }
  *before = m;
  return n;
}
// a / b for a >= 0, b > 0: 32-bit division, a quarter of the instructions, where that is enough.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}
// The units in equal, contiguous shares, one per worker (warp); a few units go to as many workers, one each.  A worker's
// number goes over the CTAs first, so that those are spread over all multiprocessors.  (Shares by how much a scheduler prefers
// its first warp to its second and third, 1.56 to 1.73 and 1.86 us per tile, made all of them end together, and later: the
// multiprocessor is as fast with the last of them alone.)
struct Shares {
  long long total;       // units
  int workers;           // that have any
  __device__ __forceinline__ Shares(long long units, int all_workers) : total(units), workers(units < all_workers ? static_cast<int>(units) : all_workers) {}
  __device__ __forceinline__ static int here() { return static_cast<int>(threadIdx.x >> 5) * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x); }
  __device__ __forceinline__ long long begin(int worker) const { return quotient(total * worker, workers); }
  __device__ __forceinline__ int of(long long unit) const { return static_cast<int>(quotient((unit + 1) * workers - 1, total)); }
};

// A place in the list: tiles t to end of item `item` of sequence b are the share's.
struct Cursor {
  int b, n, tiles, item, t, end;
  int left;                // units of the share behind this item
  long long at;            // the item's first tile in the list of tiles alone
};
// To the next item of the share that has tiles of it; t = end if there is none.
__device__ __forceinline__ void next_item(Cursor& k, const Cache4& c, const int* counts, int per_sequence, int cost) {
  while (k.left > 0) {
    k.at += k.tiles;
    if (++k.item == per_sequence) {
      k.item = 0;
      do {
        if (++k.b >= c.B) {
          k.left = k.t = k.end = 0;
          return;
        }
        k.tiles = tiles_of(c, counts, k.b);
      } while (k.tiles == 0);
      k.n = tokens_of(c, k.b);
    }
    const int units = min(k.tiles + cost, k.left);
    k.left -= units;
    k.t = 0;
    k.end = units - cost;
    if (k.end > 0) return;
  }
  k.t = k.end = 0;
}
// One warp: the cursor of the units from `from` to `to`.
__device__ __forceinline__ Cursor cursor_at(const Cache4& c, const int* counts, int per_sequence, int cost, long long from, long long to) {
  const int lane = threadIdx.x & 31;
  Cursor k;
  long long before = 0, first = 0;      // units before the sequences looked at; of the sequence
  int sequences = 0;                    // with tokens, before it
  k.b = -1;
  for (int base = 0; base < c.B && k.b < 0; base += 32) {
    const int tiles = base + lane < c.B ? tiles_of(c, counts, base + lane) : 0, units = tiles > 0 ? tiles + cost : 0;
    long long sum = units;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += u;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, (before + sum) * per_sequence > from), filled = __ballot_sync(0xffffffffu, tiles > 0);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      k.tiles = __shfl_sync(0xffffffffu, tiles, l);
      first = (before + __shfl_sync(0xffffffffu, sum, l) - (k.tiles + cost)) * per_sequence;
      sequences += __popc(filled & ((1u << l) - 1u));
      k.b = base + l;
    } else {
      before += __shfl_sync(0xffffffffu, sum, 31);
      sequences += __popc(filled);
    }
  }
  k.item = k.t = k.end = k.left = 0;
  if (k.b < 0) return k;                // only if the lengths have changed meanwhile
  k.n = tokens_of(c, k.b);
  const int length = k.tiles + cost;
  k.item = static_cast<int>(quotient(from - first, length));
  const int unit = static_cast<int>(from - first - static_cast<long long>(k.item) * length);
  const int units = static_cast<int>(min(static_cast<long long>(length - unit), to - from));
  k.at = first - static_cast<long long>(sequences) * per_sequence * cost + static_cast<long long>(k.item) * k.tiles;
  k.t = max(unit - cost, 0);
  k.end = max(unit + units - cost, 0);
  k.left = static_cast<int>(to - from) - units;
  if (k.t >= k.end) next_item(k, c, counts, per_sequence, cost);
  return k;
}

// ------------------------------------------------------------------ query rows
// Row r of an item is query token r / group of head (r % group) of the K/V head's query heads.
struct Rows {
  int group, count;    // query heads per K/V head; rows = group * S
};

// The B fragments of 8 NT query rows, each row divided by a power of two so that its largest element is about 2^10
// (fp16 then holds bf16's numbers as well), the sums of its groups and the factor that its sums are scores by.
template <int D, int NT>
struct Query {
  static constexpr int G = D / 32;
  uint32_t frag[NT][G][4];
  // Sums of the groups times 2^-9, as three numbers of the cache's type each: B fragments of the product with the
  // minima, whose k index runs over (part, group).
  static constexpr int kSumMmas = (3 * G + 7) / 8;
  uint32_t sums[NT][kSumMmas];
  float factor[NT][2];      // > 0, log2 units
  int last[NT][2];          // last visible slot
  int last_all;             // slots up to here are visible to every row
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
        const uint4 v = *reinterpret_cast<const uint4*>(src + 32 * w);
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
    const float down = copysignf(__uint_as_float(static_cast<uint32_t>(127 - e) << 23), a.sm_scale);   // 2^-e, and the scale's sign
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    float rest[G];
#pragma unroll
    for (int w = 0; w < G; ++w) {
      float sum = 0.f;   // of the group
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
      rest[w] = sum * 0.001953125f;
    }
    // every lane has numbers 2 c, 2 c + 1 of each eight
#pragma unroll
    for (int k = 0; k < Query<D, NT>::kSumMmas; ++k) f.sums[nt][k] = 0u;
#pragma unroll
    for (int part = 0; part < 3; ++part) {
#pragma unroll
      for (int w = 0; w < G; w += 2) {
        const uint32_t pair = from_f32x2<kBf16>(rest[w], rest[w + 1]);
        const float2 taken = to_f32x2<kBf16>(pair);
        rest[w] -= taken.x;
        rest[w + 1] -= taken.y;
        const int at = part * G + w;                   // k index of the pair
        if (2 * q4 == (at & 7)) f.sums[nt][at >> 3] = pair;
      }
    }
    const float factor = fmaxf(up * 512.f * (fabsf(a.sm_scale) * kLog2e), 1e-37f);   // -inf times it stays -inf
    f.factor[nt][0] = __shfl_sync(0xffffffffu, factor, 8 * q4);
    f.factor[nt][1] = __shfl_sync(0xffffffffu, factor, 8 * q4 + 4);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = row0 + 8 * nt + 2 * q4 + j, i = r / rows.group;
      f.last[nt][j] = r >= rows.count ? INT_MAX : i < count ? n - count + i : -1;   // rows that do not exist: whatever is cheap
    }
  }
  int all = INT_MAX;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) all = min(all, min(f.last[nt][0], f.last[nt][1]));
  f.last_all = __reduce_min_sync(0xffffffffu, all);
}

// ------------------------------------------------------------------ one block of 16 tokens
// Scores of tokens (g, g + 8) (g = lane / 4) and query rows (2 c, 2 c + 1) from the records at `rec`, but for the
// rows' factors.
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
  // the minima's part: groups (2 c, 2 c + 1) of either token, in every place of the k index that stands for them
  const int w2 = (2 * q4) % G;
  const uint2 ml = *reinterpret_cast<const uint2*>(lo + R::kKPairs + 4 * w2), mh = *reinterpret_cast<const uint2*>(hi + R::kKPairs + 4 * w2);
  const uint32_t m_lo = __byte_perm(ml.x, ml.y, 0x7632), m_hi = __byte_perm(mh.x, mh.y, 0x7632);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s[nt][j] = 0.f;
#pragma unroll
    for (int k = 0; k < Query<D, NT>::kSumMmas; ++k) mma_own_k8<kBf16>(s[nt], m_lo, m_hi, f.sums[nt][k]);
  }
#pragma unroll
  for (int w = 0; w < G; ++w) {
    const uint32_t a8 = kl[w] >> 8, b8 = kh[w] >> 8;
    // codes count 2^-24, the sums 2^-9
    const float sl = scale_of<kBf16>(pl[w], kBf16 ? 0x4700 : 0x7800), sh = scale_of<kBf16>(ph[w], kBf16 ? 0x4700 : 0x7800);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float acc[4];
      mma_f16_first(acc, kl[w] & 0x000f000fu, kh[w] & 0x000f000fu, a8 & 0x000f000fu, b8 & 0x000f000fu, f.frag[nt][w][0], f.frag[nt][w][1]);
      mma_f16(acc, kl[w] & 0x00f000f0u, kh[w] & 0x00f000f0u, a8 & 0x00f000f0u, b8 & 0x00f000f0u, f.frag[nt][w][2], f.frag[nt][w][3]);
      s[nt][0] = fmaf(sl, acc[0], s[nt][0]);
      s[nt][1] = fmaf(sl, acc[1], s[nt][1]);
      s[nt][2] = fmaf(sh, acc[2], s[nt][2]);
      s[nt][3] = fmaf(sh, acc[3], s[nt][3]);
    }
  }
}

// The sums of one piece of an item.  sum p s u + sum p m is taken as sum P (u - 8) + sum p (m + 8 s), P = fp16(p s): the
// rounding of P then shows times u - 8 instead of u, and neither it nor an MMA's own (which cuts its sums off, at 2^-24 of what
// its operands' exponents allow) comes up against a sum that is mostly the codes' middle.  With u * 2^-24 as the operand
// here, too, results were off by 4.5e-4 over 60000 tokens, with u - 8 by 2.8e-4 (fp16, whose own rounding is 2.1e-4).
// The last sum (`mids`) comes out of MMAs of its own, whose rows w and w + 8 are the minima and the scales of group w as they
// are stored.  They take p as its 16-bit rounding and what that leaves, 16 bits of it or more: the sum that the result is divided
// by has all 32, and V rows that have much in common would not come back as that (with the first part alone bf16 results
// were off by 1.71e-3 for 1.67e-3, 1.67e-3 of it their own rounding; 64 sequences of 1 to 8192 tokens 85.7 us for 86.9).
template <int D, int NT>
struct Sums {
  static constexpr int G = D / 32;
  float o[2 * G][NT][4];       // tile 2 w + t: dims 32 w + 4 g + 2 t and + 1, times 2^-9 over `unit`
  float mids[NT][4];           // sum p m of group g % G, rows 2 c, 2 c + 1, then sum p s
  float l[NT][2], ref[NT][2];
  float unit;                  // power of two that s is divided by
  uint32_t per_unit;           // 1 / unit, a 16-bit number of the cache's type; bf16: above it the unit that others are held against (raise)
  uint32_t unit_limit;         // 16-bit pattern of the scale from which on it is raised
};
// 1 / unit has to be a number of the cache's type: 2^-15 and 2^-100.  Scales below that are fp16's subnormal ones.
template <bool kBf16>
constexpr float kLeastUnit = kBf16 ? 7.888609052210118e-31f : 3.0517578125e-5f;
constexpr float kNoScore = -3.4028234663852886e38f;    // reference of a row that has seen nothing

template <int D, int NT, bool kBf16>
__device__ __forceinline__ void clear(Sums<D, NT>& x) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x.mids[nt][i] = 0.f;
#pragma unroll
    for (int j = 0; j < 2 * (D / 32); ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) x.o[j][nt][i] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x.l[nt][i] = 0.f;
      x.ref[nt][i] = kNoScore;
    }
  }
  x.unit = kLeastUnit<kBf16>;
  x.per_unit = from_f32<kBf16>(1.f / kLeastUnit<kBf16>);
  x.unit_limit = from_f32<kBf16>(kLeastUnit<kBf16> * kRaiseScale);
}

// Tokens of a block whose V pairs are NaN: a row that gives one of them weight gets NaN for the group, and the pairs
// are made zeros, so that rows which do not see the token do not see NaN either.
template <int D, int NT, bool kBf16>
__device__ __noinline__ void defuse_block(uint8_t* rec, const float* p, float* mids) {
  using R = Record<D>;
  constexpr int G = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  for (int token = 0; token < 16; ++token) {
    const uint32_t pair = *reinterpret_cast<const uint32_t*>(rec + token * R::kBytes + R::kVPairs + 4 * (g % G));
    const float2 sm = to_f32x2<kBf16>(pair);
    const bool nan = !(fabsf(sm.x) < INFINITY && fabsf(sm.y) < INFINITY);
    for (int nt = 0; nt < NT; ++nt)
      for (int i = 0; i < 2; ++i) {
        const float w = __shfl_sync(0xffffffffu, p[4 * nt + 2 * (token >> 3) + i], 4 * (token & 7) + q4);
        if (nan && w != 0.f) mids[4 * nt + i] = __int_as_float(0x7fffffff);
      }
    __syncwarp();
    if (nan && q4 == 0 && g < G) *reinterpret_cast<uint32_t*>(rec + token * R::kBytes + R::kVPairs + 4 * g) = 0u;
  }
  __syncwarp();
}

// The second product of 16 tokens: p of tokens (g, g + 8).
template <int D, int NT, bool kBf16>
__device__ __forceinline__ void block_output(Sums<D, NT>& x, const float (&p)[NT][4], const uint8_t* rec) {
  using R = Record<D>;
  constexpr int G = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  constexpr int kWords = G / 2;                  // 32-bit words of one token's V codes in a lane
  uint32_t v[4][kWords], mid[4], pl[G], ph[G];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint8_t* token = rec + (2 * q4 + (j & 1) + 8 * (j >> 1)) * R::kBytes;
    const uint8_t* at = token + R::kVCodes + g * (D / 16);
    if constexpr (kWords == 1) {
      v[j][0] = *reinterpret_cast<const uint32_t*>(at);
    } else if constexpr (kWords == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(at);
      v[j][0] = u.x, v[j][1] = u.y;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(at);
      v[j][0] = u.x, v[j][1] = u.y, v[j][2] = u.z, v[j][3] = u.w;
    }
    mid[j] = *reinterpret_cast<const uint32_t*>(token + R::kVPairs + 4 * (g % G));
  }
  const uint8_t* lo = rec + g * R::kBytes + R::kVPairs;
  const uint8_t* hi = lo + 8 * R::kBytes;
  if constexpr (G == 2) {
    const uint2 y = *reinterpret_cast<const uint2*>(lo), z = *reinterpret_cast<const uint2*>(hi);
    pl[0] = y.x, pl[1] = y.y, ph[0] = z.x, ph[1] = z.y;
  } else {
#pragma unroll
    for (int w = 0; w < G; w += 4) {
      const uint4 y = *reinterpret_cast<const uint4*>(lo + 4 * w), z = *reinterpret_cast<const uint4*>(hi + 4 * w);
      pl[w] = y.x, pl[w + 1] = y.y, pl[w + 2] = y.z, pl[w + 3] = y.w;
      ph[w] = z.x, ph[w + 1] = z.y, ph[w + 2] = z.z, ph[w + 3] = z.w;
    }
  }
  // rows of minima, then rows of scales
  const uint32_t m_lo = __byte_perm(mid[0], mid[1], 0x7632), s_lo = __byte_perm(mid[0], mid[1], 0x5410);
  const uint32_t m_hi = __byte_perm(mid[2], mid[3], 0x7632), s_hi = __byte_perm(mid[2], mid[3], 0x5410);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const uint32_t p_lo = from_f32x2<kBf16>(p[nt][0], p[nt][1]), p_hi = from_f32x2<kBf16>(p[nt][2], p[nt][3]);
    const float2 t_lo = to_f32x2<kBf16>(p_lo), t_hi = to_f32x2<kBf16>(p_hi);
    mma_own<kBf16>(x.mids[nt], m_lo, s_lo, m_hi, s_hi, transpose_8x8(p_lo), transpose_8x8(p_hi));
    mma_own<kBf16>(x.mids[nt], m_lo, s_lo, m_hi, s_hi, transpose_8x8(from_f32x2<kBf16>(p[nt][0] - t_lo.x, p[nt][1] - t_lo.y)),
                   transpose_8x8(from_f32x2<kBf16>(p[nt][2] - t_hi.x, p[nt][3] - t_hi.y)));
  }
#pragma unroll
  for (int w = 0; w < G; ++w) {
    // the half words of group w: low half token 2 c (2 c + 8), high half the token behind it
    const uint32_t pick = (w & 1) ? 0x7632u : 0x5410u;
    const uint32_t y = __byte_perm(v[0][w / 2], v[1][w / 2], pick), z = __byte_perm(v[2][w / 2], v[3][w / 2], pick);
    const uint32_t y8 = y >> 8, z8 = z >> 8;
    const uint32_t ya = centred<false>(y & 0x000f000fu), yb = centred<true>(y & 0x00f000f0u), za = centred<false>(z & 0x000f000fu),
                   zb = centred<true>(z & 0x00f000f0u);
    const uint32_t yc = centred<false>(y8 & 0x000f000fu), yd = centred<true>(y8 & 0x00f000f0u), zc = centred<false>(z8 & 0x000f000fu),
                   zd = centred<true>(z8 & 0x00f000f0u);
    const float sl = scale_of<kBf16>(pl[w], static_cast<uint16_t>(x.per_unit)), sh = scale_of<kBf16>(ph[w], static_cast<uint16_t>(x.per_unit));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t pl2 = from_f32x2<false>(p[nt][0] * sl, p[nt][1] * sl), ph2 = from_f32x2<false>(p[nt][2] * sh, p[nt][3] * sh);
      const uint32_t b0 = transpose_8x8(pl2), b1 = transpose_8x8(ph2);
      mma_f16(x.o[2 * w][nt], ya, yb, za, zb, b0, b1);
      mma_f16(x.o[2 * w + 1][nt], yc, yd, zc, zd, b0, b1);
    }
  }
}

// What the widest finite scale of a lane's share of a tile is (see one_tile), where one that is not finite hides it.
template <int D, bool kBf16>
__device__ __noinline__ uint32_t widest_finite(const uint8_t* rec) {
  using R = Record<D>;
  constexpr int G = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  uint32_t widest = 0;
  for (int token = g; token < tile_tokens(D); token += 8)
    for (int w = 0; w < (G + 3) / 4; ++w) {
      const uint32_t scale = *reinterpret_cast<const uint16_t*>(rec + token * R::kBytes + R::kVPairs + 4 * ((q4 + 4 * w) % G));
      if (scale < (kBf16 ? 0x7f80u : 0x7c00u)) widest = max(widest, scale);
    }
  return widest;
}

// The narrowest scale of a tile that is one (a group without a range has none); infinity: there is none.
template <int D, bool kBf16>
__device__ __noinline__ float narrowest(const uint8_t* rec) {
  using R = Record<D>;
  constexpr int G = D / 32;
  constexpr uint32_t kInf = kBf16 ? 0x7f80u : 0x7c00u;
  uint32_t least = kInf;               // as integers, less one: zero comes last
  for (int token = threadIdx.x & 31; token < tile_tokens(D); token += 32)
#pragma unroll
    for (int w = 0; w < G; w += 2) {
      const uint2 pairs = *reinterpret_cast<const uint2*>(rec + token * R::kBytes + R::kVPairs + 4 * w);
      least = min(least, min((pairs.x & 0xffffu) - 1u, (pairs.y & 0xffffu) - 1u));
    }
  least = __reduce_min_sync(0xffffffffu, least);
  return least >= kInf - 1u ? INFINITY : to_f32<kBf16>(static_cast<uint16_t>(least + 1u));
}
// log2 of the largest p * s of 16 tokens per query row, from log2 p of tokens (g, g + 8), against what `most` holds.
template <int D, int NT, bool kBf16>
__device__ __noinline__ void largest_products(const uint8_t* rec, const float* p, float* most) {
  using R = Record<D>;
  constexpr int G = D / 32;
  const int g = (threadIdx.x & 31) >> 2;
  for (int i = 0; i < 2; ++i) {
    float widest = 0.f;
    for (int w = 0; w < G; ++w) {
      const float scale = to_f32<kBf16>(*reinterpret_cast<const uint16_t*>(rec + (g + 8 * i) * R::kBytes + R::kVPairs + 4 * w));
      if (scale < INFINITY) widest = fmaxf(widest, scale);
    }
    for (int nt = 0; nt < NT; ++nt)
      for (int j = 0; j < 2; ++j) most[2 * nt + j] = fmaxf(most[2 * nt + j], p[4 * nt + 2 * i + j] + __log2f(widest));
  }
}

// Raises the references of the rows to the largest score of a tile, and the unit to its widest scale.  Both in one
// place: with a branch each the sums were copied from register to register in every tile (16 of 344 instructions per 16
// tokens).
//
// The unit is all rows', and a row whose own scales are far below it has its products rounded away: fp16's range from
// 2^13 down to 2^-24 is enough for scales that are fp16 numbers themselves, those of bf16 can be 2^40 apart, in a token that the
// row does not see.  So in bf16 a scale more than kFar above the narrowest of the first tile raises the unit only to where each
// row's largest product of the tile is still 2^0; a row with larger products than fp16 holds gets a higher reference instead.
template <int D, int NT, bool kBf16>
__device__ __forceinline__ void raise(Sums<D, NT>& x, const float (&top)[NT][2], uint32_t widest, const float (&s)[tile_tokens(D) / 16][NT][4],
                                      const Query<D, NT>& f, const uint8_t* rec) {
  auto power_below = [](float v) { return __uint_as_float(__float_as_uint(v) & 0x7f800000u); };
  const float scale = to_f32<kBf16>(static_cast<uint16_t>(__reduce_max_sync(0xffffffffu, widest)));   // finite
  // the power of two below it, where it is above what the unit is for
  float unit = scale > x.unit * kRaiseScale ? power_below(scale) : x.unit;
  float ref[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float m = top[nt][i];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      ref[nt][i] = m > x.ref[nt][i] + kRaise ? m - kHeadroom : x.ref[nt][i];
    }
  if constexpr (kBf16) {
    if (unit > x.unit) {
      float base = __uint_as_float(x.per_unit & 0xffff0000u);
      if (base == 0.f) base = power_below(narrowest<D, kBf16>(rec));
      if (unit > base * kFar) {
        float most[2 * NT], least = INFINITY;
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) most[i] = -INFINITY;
        for (int k = 0; k < tile_tokens(D) / 16; ++k) {
          float p[4 * NT];
#pragma unroll
          for (int j = 0; j < 4 * NT; ++j) {
            float score = s[0][j / 4][j % 4];
#pragma unroll
            for (int t = 1; t < tile_tokens(D) / 16; ++t)
              if (t == k) score = s[t][j / 4][j % 4];
            p[j] = fmaf(score, f.factor[j / 4][j & 1], -ref[j / 4][j & 1]);
          }
          largest_products<D, NT, kBf16>(rec + 16 * k * Record<D>::kBytes, p, most);
        }
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
          for (int d = 4; d < 32; d <<= 1) most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], d));
          if (most[i] > -INFINITY) least = fminf(least, most[i]);  // a row that sees something
        }
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, 1));
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, 2));
        const int exponent = static_cast<int>(floorf(fminf(fmaxf(least, -100.f), 125.f)));
        // no less than what makes scale / unit a 32-bit number
        unit = fmaxf(fmaxf(x.unit, unit * 7.5231638452626401e-37f), fminf(unit, fmaxf(base, __uint_as_float(static_cast<uint32_t>(127 + exponent) << 23))));
        const float log2_unit = static_cast<float>(static_cast<int>(__float_as_uint(unit) >> 23) - 127);
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) ref[i / 2][i % 2] += fmaxf(ceilf(most[i] - log2_unit - 13.f), 0.f);
        base = unit;
      }
      x.per_unit = __float_as_uint(base);
    }
  }
  const float by_unit = x.unit / unit;
  x.unit = unit;
  x.per_unit = (kBf16 ? x.per_unit & 0xffff0000u : 0u) | from_f32<kBf16>(1.f / unit);
  x.unit_limit = from_f32<kBf16>(unit * kRaiseScale);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float by = ex2(x.ref[nt][i] - ref[nt][i]), by_both = by * by_unit;
      x.ref[nt][i] = ref[nt][i];
      x.l[nt][i] *= by;
      x.mids[nt][i] *= by;
      x.mids[nt][i + 2] *= by;
#pragma unroll
      for (int j = 0; j < 2 * (D / 32); ++j) {
        x.o[j][nt][i] *= by_both;
        x.o[j][nt][i + 2] *= by_both;
      }
    }
}

// One tile at `rec`, whose first slot is `slot`.  scores: where the tile's scores are kept, null: nowhere.
// True if `rec` was written to.
template <int D, int NT, bool kBf16>
__device__ __forceinline__ bool one_tile(Sums<D, NT>& x, const Query<D, NT>& f, uint8_t* rec, int slot, float* scores, int score_rows) {
  using R = Record<D>;
  constexpr int G = D / 32, kTile = tile_tokens(D), kBlocks = kTile / 16;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  float s[kBlocks][NT][4];
#pragma unroll
  for (int k = 0; k < kBlocks; ++k) block_scores<D, NT, kBf16>(s[k], rec + 16 * k * R::kBytes, f);
  if (slot + kTile - 1 > f.last_all) {
#pragma unroll
    for (int k = 0; k < kBlocks; ++k)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (slot + 16 * k + g + 8 * (j >> 1) > f.last[nt][j & 1]) s[k][nt][j] = -INFINITY;
  }
  bool higher = false;
  float top[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float most = fmaxf(s[0][nt][i], s[0][nt][i + 2]);
#pragma unroll
      for (int k = 1; k < kBlocks; ++k) most = max3(most, s[k][nt][i], s[k][nt][i + 2]);
      top[nt][i] = most * f.factor[nt][i];
      higher |= top[nt][i] > x.ref[nt][i] + kRaise;
    }
  // a scale much above all before: each lane looks at its share of the tile's (as integers, which their bits order like)
  uint32_t widest = 0;
#pragma unroll
  for (int i = 0; i < 2 * kBlocks; ++i)
#pragma unroll
    for (int w = 0; w < (G + 3) / 4; ++w)
      widest = max(widest, *reinterpret_cast<const uint16_t*>(rec + (g + 8 * i) * R::kBytes + R::kVPairs + 4 * ((q4 + 4 * w) % G)) + 0u);
  bool odd = false;
  if (__any_sync(0xffffffffu, higher || widest > x.unit_limit)) {
    odd = __any_sync(0xffffffffu, widest >= (kBf16 ? 0x7f80u : 0x7c00u));
    if (odd) widest = widest_finite<D, kBf16>(rec);
    raise<D, NT, kBf16>(x, top, widest, s, f, rec);
  }
  if (scores != nullptr) {
#pragma unroll
    for (int k = 0; k < kBlocks; ++k)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 8 * nt + 2 * q4 + (j & 1);
          if (r < score_rows) scores[r * kTile + 16 * k + g + 8 * (j >> 1)] = s[k][nt][j] * f.factor[nt][j & 1];
        }
  }
#pragma unroll
  for (int k = 0; k < kBlocks; ++k)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[k][nt][j] = ex2(fmaf(s[k][nt][j], f.factor[nt][j & 1], -x.ref[nt][j & 1]));
        x.l[nt][j & 1] += s[k][nt][j];
      }
  if (odd) {
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      float weights[4 * NT], mids[4 * NT];
#pragma unroll
      for (int j = 0; j < 4 * NT; ++j) weights[j] = s[k][j / 4][j % 4], mids[j] = x.mids[j / 4][j % 4];
      defuse_block<D, NT, kBf16>(rec + 16 * k * R::kBytes, weights, mids);
#pragma unroll
      for (int j = 0; j < 4 * NT; ++j) x.mids[j / 4][j % 4] = mids[j];
    }
  }
#pragma unroll
  for (int k = 0; k < kBlocks; ++k) block_output<D, NT, kBf16>(x, s[k], rec + 16 * k * R::kBytes);
  return odd;
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
  auto whole = [&](float v) { return v * 512.f * x.unit; };
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // what goes to every dim of a group: its mids, which lane 4 w + q4 has
      float l = x.l[nt][i], m[G];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
#pragma unroll
      for (int w = 0; w < G; ++w) m[w] = __shfl_sync(0xffffffffu, fmaf(8.f, x.mids[nt][i + 2], x.mids[nt][i]), 4 * w + q4);
      const int r = 8 * nt + 2 * q4 + i, row = row0 + r;
      if (row < rows.count) {
        if (piece != nullptr) {
          float* dst = piece + r * (D + 2);
#pragma unroll
          for (int w = 0; w < G; ++w) {
            *reinterpret_cast<float2*>(dst + 32 * w + 4 * g) = make_float2(whole(x.o[2 * w][nt][i]) + m[w], whole(x.o[2 * w][nt][i + 2]) + m[w]);
            *reinterpret_cast<float2*>(dst + 32 * w + 4 * g + 2) =
                make_float2(whole(x.o[2 * w + 1][nt][i]) + m[w], whole(x.o[2 * w + 1][nt][i + 2]) + m[w]);
          }
          if (g == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(x.ref[nt][i], l);
        } else {
          const int t = row / rows.group, hq = h * rows.group + row - t * rows.group;
          const float inv = l == 0.f ? 0.f : 1.f / l;      // a row that sees nothing is zero
          uint16_t* dst = static_cast<uint16_t*>(a.o) + b * a.o_stride[0] + hq * a.o_stride[1] + t * a.o_stride[2];
#pragma unroll
          for (int w = 0; w < G; ++w)
            *reinterpret_cast<uint2*>(dst + 32 * w + 4 * g) =
                make_uint2(from_f32x2<kBf16>((whole(x.o[2 * w][nt][i]) + m[w]) * inv, (whole(x.o[2 * w][nt][i + 2]) + m[w]) * inv),
                           from_f32x2<kBf16>((whole(x.o[2 * w + 1][nt][i]) + m[w]) * inv, (whole(x.o[2 * w + 1][nt][i + 2]) + m[w]) * inv));
          if (g == 0 && a.lse != nullptr)
            a.lse[(static_cast<int64_t>(b) * a.Hq + hq) * a.S + t] = l == 0.f ? -INFINITY : (x.ref[nt][i] + __log2f(l)) * kLn2;
        }
      }
    }
  }
}

// Every warp works for itself: a ring of tiles in shared memory, which its first lane fills with bulk copies as soon
// as the warp is done with a slot, across the items of its share.
template <int D, int NT, bool kBf16>
__global__ void __launch_bounds__((Shape<D, NT>::kThreads), 1) cache4_attention_kernel(const Cache4 c, const Cache4Attention a, const Rows rows,
                                                                                        const int row_blocks, const bool keep, const unsigned long long wait_limit_ns,
                                                                                        const int test_drop_load) {
  using R = Record<D>;
  using Sh = Shape<D, NT>;
  constexpr int kTile = Sh::kTile;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t full_bar[Sh::kWarps * Sh::kStages];
  __shared__ int abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < Sh::kWarps * Sh::kStages) mbar_init(smem_u32(&full_bar[threadIdx.x]), 1);
  if (threadIdx.x == 0) abort_word = 0;
  fence_barrier_init();
  fence_proxy_async();
  __syncthreads();
  // The kernels behind this one read lengths and pages before it is done: they may not start before the ones in front
  // of it are.
  griddep_wait();
  griddep_launch_dependents();
  const int per_sequence = c.H * row_blocks;
  long long none;
  const long long total = all_units(c, a.counts, kItemCost, 0, &none) * per_sequence;
  const Shares shares(total, gridDim.x * Sh::kWarps);
  const int worker = shares.here();
  if (worker >= shares.workers) return;
  Cursor use = cursor_at(c, a.counts, per_sequence, kItemCost, shares.begin(worker), shares.begin(worker + 1));
  if (use.t >= use.end) return;            // nothing but an item's cost
  Cursor load = use;
  uint8_t* const my_ring = ring + warp * Sh::kStages * Sh::kSlotBytes;
  const uint32_t my_bar = smem_u32(&full_bar[warp * Sh::kStages]);
  const int mask = (1 << c.page_shift) - 1;
  // The pieces window .. window + 31 of the item in `load`, one per lane: its page (-1: none) and address; the pages
  // behind them are on their way.
  int window = 0, pages = -1, pages_next = -1;
  const uint8_t* piece_at = nullptr;
  uint32_t there = 0;                      // lanes that have a page
  uint32_t have = 0;                       // a bit per piece of every slot: asked for
  constexpr uint32_t kAll = (1u << Sh::kPieces) - 1u;
  int drop = test_drop_load + 1;
  auto page_of = [&](int piece) {
    const int slot = piece * 16;
    return slot < load.n ? c.table[static_cast<int64_t>(load.b) * c.table_stride + (slot >> c.page_shift)] : -1;
  };
  auto open_window = [&](int first, int known) {
    window = first;
    pages = known;
    const bool used = (window + lane) * 16 < load.n, ok = used && static_cast<unsigned>(pages) < static_cast<unsigned>(c.pages);
    if (used && !ok) report_bad_index(c.status, kTagCachePage);
    there = __ballot_sync(0xffffffffu, ok);
    piece_at = c.kv + load.item / row_blocks * c.kv_stride[1] + (ok ? pages : 0) * c.kv_stride[0] +
               static_cast<int64_t>((window + lane) * 16 & mask) * R::kBytes;
    pages_next = page_of(window + 32 + lane);
  };
  open_window(load.t * Sh::kPieces, page_of(load.t * Sh::kPieces + lane));
  auto issue = [&](int stage) {
    const int off = load.t * Sh::kPieces - window;
    const uint32_t asked = (there >> off) & kAll;
    have = (have & ~(kAll << (Sh::kPieces * stage))) | asked << (Sh::kPieces * stage);
    const uint32_t bar = my_bar + 8 * stage;
    if (--drop == 0) {                     // test hook: neither the load nor the arrival that announces it
      if (++load.t == load.end) next_item(load, c, a.counts, per_sequence, kItemCost);
      return;
    }
    if (lane == 0) mbar_arrive_expect_tx(bar, __popc(asked) * Sh::kPieceBytes);
    const int i = lane - off;
    if (static_cast<unsigned>(i) < Sh::kPieces && ((there >> lane) & 1))
      bulk_load(smem_u32(my_ring + stage * Sh::kSlotBytes) + i * Sh::kPieceBytes, piece_at, bar, Sh::kPieceBytes);
    if (++load.t == load.end) {
      const int b = load.b;
      next_item(load, c, a.counts, per_sequence, kItemCost);
      // the next head of a short sequence has the same pages
      if (load.t < load.end) open_window(0, load.b == b && window == 0 ? pages : page_of(lane));
    } else if (off + Sh::kPieces == 32) {
      open_window(window + 32, pages_next);
    }
  };

  const int score_rows = min(8 * NT, rows.count);     // of a tile; as many as an item has
  float* const kept = keep ? a.scores : nullptr;
  for (int i = 0; i < Sh::kStages && load.t < load.end; ++i) issue(i);
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  while (use.t < use.end) {
    // one piece: the tiles of one item that belong to this share
    const int b = use.b, t0 = use.t, tiles = use.tiles, h = use.item / row_blocks, row0 = (use.item - h * row_blocks) * 8 * NT, n = use.n;
    const int t1 = use.end;
    Query<D, NT> f;
    load_query<D, NT, kBf16>(f, c, a, rows, b, h, row0, n);
    Sums<D, NT> x;
    clear<D, NT, kBf16>(x);
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      ok = mbar_wait_warp(my_bar + 8 * stage, phase, &abort_word, wait_limit_ns, kTagCache4Load);
      if (!ok) break;
      uint8_t* const slot = my_ring + stage * Sh::kSlotBytes;
      // what is not there, tokens behind the last one and pages that do not exist, is made zeros
      const int left = min(n - t * kTile, kTile);
      const uint32_t asked = (have >> (Sh::kPieces * stage)) & kAll;
      const bool patch = left < kTile || asked != kAll;
      if (patch) {
        for (int i = lane; i < kTile * (R::kBytes / 16); i += 32) {
          const int token = i / (R::kBytes / 16);
          if (token >= left || !((asked >> (token >> 4)) & 1)) *reinterpret_cast<uint4*>(slot + 16 * i) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      float* scores = kept != nullptr ? kept + (use.at + t) * score_rows * kTile : nullptr;
      const bool written = one_tile<D, NT, kBf16>(x, f, slot, t * kTile, scores, score_rows);
      if (patch || written) fence_proxy_async();      // before a copy writes where this warp has written
      __syncwarp();
      if (load.t < load.end) issue(stage);
      if (++stage == Sh::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!ok) break;
    float* piece = nullptr;
    if (t0 > 0 || t1 < tiles) piece = a.pieces + (worker * 2ll + (t0 == 0)) * piece_floats<D, NT>();
    store_sums<D, NT, kBf16>(x, a, rows, b, h, row0, piece);
    next_item(use, c, a.counts, per_sequence, kItemCost);
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

// A CTA has an item's rows from blockIdx.y * rows_each on: it joins the item's pieces where there are several, and
// answers for items without tokens.  The pieces are taken in an order that does not depend on timing.
template <int D, int NT, bool kBf16>
__global__ void __launch_bounds__(kJoinMost) cache4_join_kernel(const Cache4 c, const Cache4Attention a, const Rows rows, const int row_blocks,
                                                                const int all_workers, const int rows_each) {
  constexpr int kEach = D / 32;
  __shared__ float part[kJoinMost / 32][D];
  __shared__ float2 sums[kJoinMost / 32];
  fence_ahead();
  const int item = blockIdx.x % (c.H * row_blocks), b = blockIdx.x / (c.H * row_blocks), h = item / row_blocks;
  const int from = blockIdx.y * rows_each, row0 = (item - h * row_blocks) * 8 * NT + from;
  const int count = min(min(rows_each, 8 * NT - from), rows.count - row0);   // rows of this CTA
  if (count <= 0) {
    griddep_wait();              // no CTA ends before the kernel in front does
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int tiles = tiles_of(c, a.counts, b);
  auto answer = [&](int row, int64_t* at_lse) {
    const int t = row / rows.group, hq = h * rows.group + row - t * rows.group;
    *at_lse = (static_cast<int64_t>(b) * a.Hq + hq) * a.S + t;
    return static_cast<uint16_t*>(a.o) + b * a.o_stride[0] + hq * a.o_stride[1] + t * a.o_stride[2];
  };
  if (tiles == 0) {
    griddep_wait();
    griddep_launch_dependents();
    for (int r = warp; r < count; r += warps) {
      int64_t at_lse;
      uint16_t* dst = answer(row0 + r, &at_lse);
      for (int d = lane; d < D; d += 32) dst[d] = 0;
      if (lane == 0 && a.lse != nullptr) a.lse[at_lse] = -INFINITY;
    }
    return;
  }
  const int per_sequence = c.H * row_blocks;
  long long before;
  const long long total = all_units(c, a.counts, kItemCost, b, &before) * per_sequence;
  const Shares shares(total, all_workers);
  const long long first = before * per_sequence + static_cast<long long>(item) * (tiles + kItemCost) + kItemCost;   // unit of its first tile
  const int w0 = shares.of(first), pieces = shares.of(first + tiles - 1) - w0 + 1;
  // lengths were there before the first kernel started, its pieces are now
  griddep_wait();
  griddep_launch_dependents();
  if (pieces == 1) return;                    // answered already
  // the warps in teams, one per row, as far as they go
  const int teams = min(count, warps), members = warps / teams, team = warp % teams, member = warp / teams;
  for (int r0 = 0; r0 < count; r0 += teams) {
    const int r = r0 + team;
    const bool busy = r < count && member < members;
    if (busy) {
      auto piece_of = [&](int i) {            // the first one is its worker's last item, the others their workers' first
        return a.pieces + ((w0 + i) * 2ll + (i == 0)) * piece_floats<D, NT>() + (from + r) * (D + 2);
      };
      float ref = kNoScore, l = 0.f, sum[kEach];
#pragma unroll
      for (int j = 0; j < kEach; ++j) sum[j] = 0.f;
      // 32 pieces at a time: references and weights one piece per lane, the sums piece by piece
      for (int i0 = member; i0 < pieces; i0 += 32 * members) {
        const int mine = i0 + lane * members;
        const float2 ml = mine < pieces ? *reinterpret_cast<const float2*>(piece_of(mine) + D) : make_float2(kNoScore, 0.f);
        float next[kEach];                    // of the first piece, asked for at once: where there are few it is the only one
#pragma unroll
        for (int j = 0; j < kEach; ++j) next[j] = piece_of(i0)[lane + 32 * j];
        float top = ml.x;
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        top = fmaxf(top, ref);
        const float before = ex2(ref - top), by = ex2(ml.x - top);
        ref = top;
        l = l * before + by * ml.y;           // of this lane's pieces
#pragma unroll
        for (int j = 0; j < kEach; ++j) sum[j] *= before;
        const int here = min(32, (pieces - i0 + members - 1) / members);
        const float share0 = __shfl_sync(0xffffffffu, by, 0);
#pragma unroll
        for (int j = 0; j < kEach; ++j) sum[j] = fmaf(share0, next[j], sum[j]);
#pragma unroll 8
        for (int k = 1; k < here; ++k) {
          const float* p = piece_of(i0 + k * members);
          const float share = __shfl_sync(0xffffffffu, by, k);
#pragma unroll
          for (int j = 0; j < kEach; ++j) sum[j] = fmaf(share, p[lane + 32 * j], sum[j]);
        }
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
#pragma unroll
      for (int j = 0; j < kEach; ++j) part[warp][lane + 32 * j] = sum[j];
      if (lane == 0) sums[warp] = make_float2(ref, l);
    }
    __syncthreads();
    if (busy && member == 0) {
      float ref = kNoScore, o[kEach], l = 0.f;
      for (int m = 0; m < members; ++m) ref = fmaxf(ref, sums[team + m * teams].x);
#pragma unroll
      for (int j = 0; j < kEach; ++j) o[j] = 0.f;
      for (int m = 0; m < members; ++m) {
        const float2 ml = sums[team + m * teams];
        const float by = ex2(ml.x - ref);
        l += by * ml.y;
#pragma unroll
        for (int j = 0; j < kEach; ++j) o[j] += by * part[team + m * teams][lane + 32 * j];
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      int64_t at_lse;
      uint16_t* dst = answer(row0 + r, &at_lse);
#pragma unroll
      for (int j = 0; j < kEach; ++j) dst[lane + 32 * j] = from_f32<kBf16>(o[j] * inv);
      if (lane == 0 && a.lse != nullptr) a.lse[at_lse] = l == 0.f ? -INFINITY : (ref + __log2f(l)) * kLn2;
    }
    __syncthreads();
  }
}

// The weights: every token's softmax weights over all query rows of its K/V head, added to weight[].  A token belongs to
// one warp, so nothing is added twice at once and the order is fixed.  This one reads the scores that the attention
// kernel has kept, 4 bytes per row and token: 128 tokens per warp at a time, four per lane.  What bounds it is how much of
// that is on its way at once: 2 sequences of 131072 tokens, 8 heads of 8 rows, 18 us (67 MB of scores, mostly from L2, and
// 17 of weights: 4.7 TB/s; 4 bytes per load and page numbers looked up when they are needed: 29 us).
template <int kTile>
__global__ void __launch_bounds__(kWeightThreads) cache4_weight_kernel(const Cache4 c, const Cache4Attention a, const Rows rows) {
  griddep_launch_dependents();
  fence_ahead();
  const int lane = threadIdx.x & 31;
  long long none;
  const long long total = all_units(c, a.counts, 0, 0, &none) * c.H;
  const Shares shares(total, gridDim.x * kWeightWarps);
  const int worker = shares.here();
  const bool used = worker < shares.workers;
  Cursor k;
  if (used) k = cursor_at(c, a.counts, c.H, 0, shares.begin(worker), shares.begin(worker + 1));
  griddep_wait();          // lengths were there before the first kernel started
  if (!used) return;       // behind the wait: this grid's end has to be behind that of the ones in front
  const int mask = (1 << c.page_shift) - 1;
  while (k.t < k.end) {
    // log-sum-exps of the item's rows, one per lane (there are no more than 16)
    float lse = 0.f;
    if (lane < rows.count) {
      const int t = lane / rows.group, hq = k.item * rows.group + lane - t * rows.group;
      lse = a.lse[(static_cast<int64_t>(k.b) * a.Hq + hq) * a.S + t] * kLog2e;
      if (lse == -INFINITY) lse = 0.f;                         // a row that sees nothing: its scores are -inf
    }
    // 32 tokens are a group, four of them neighbouring tokens of a lane; four groups at a time, and the page numbers of the
    // four behind them
    constexpr int kPerTile = kTile / 32, kRows = 4;
    const int groups = (k.end - k.t) * kPerTile, own = lane >> 3, quad = 4 * (lane & 7);
    auto slot_of = [&](int i) { return k.t * kTile + 32 * (i + own) + quad; };
    auto page_of = [&](int i) {
      const int slot = slot_of(i);
      return i + own < groups && slot < k.n ? c.table[k.b * c.table_stride + (slot >> c.page_shift)] : 0;
    };
    int next_page = page_of(0);
    for (int i = 0; i < groups; i += 4) {
      const int g = min(i + own, groups - 1), slot = slot_of(i), page = next_page;
      const float* scores = a.scores + (k.at + k.t + g / kPerTile) * rows.count * kTile + g % kPerTile * 32 + quad;
      int live = i + own < groups ? min(max(k.n - slot, 0), 4) : 0;
      if (page < 0 || page >= c.pages) {
        report_bad_index(c.status, kTagCachePage);
        live = 0;
      }
      float* weight = c.weight + page * c.weight_stride[0] + k.item * c.weight_stride[1] + (slot & mask);
      float old[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j) old[j] = j < live ? weight[j] : 0.f;
      if (i + 4 < groups) next_page = page_of(i + 4);
      for (int r0 = 0; r0 < rows.count; r0 += kRows) {
        float4 v[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          v[r] = r0 + r < rows.count ? *reinterpret_cast<const float4*>(scores + (r0 + r) * kTile) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float of_row = __shfl_sync(0xffffffffu, lse, r0 + r);
          sum[0] += ex2(v[r].x - of_row);
          sum[1] += ex2(v[r].y - of_row);
          sum[2] += ex2(v[r].z - of_row);
          sum[3] += ex2(v[r].w - of_row);
        }
      }
      if (__any_sync(0xffffffffu, lse != lse)) {               // a row is NaN: the tokens that it does not see are not
        sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
#pragma unroll 1
        for (int r = 0; r < rows.count; ++r) {
          const float of_row = __shfl_sync(0xffffffffu, lse, r);
          const float4 x = *reinterpret_cast<const float4*>(scores + r * kTile);
          if (x.x != -INFINITY) sum[0] += ex2(x.x - of_row);
          if (x.y != -INFINITY) sum[1] += ex2(x.y - of_row);
          if (x.z != -INFINITY) sum[2] += ex2(x.z - of_row);
          if (x.w != -INFINITY) sum[3] += ex2(x.w - of_row);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live) weight[j] = old[j] + sum[j];
    }
    next_item(k, c, a.counts, c.H, 0);
  }
}

// The same without kept scores (see keeps_scores): they are computed again from K, against the rows' log-sum-exp.
template <int D, int NT, bool kBf16>
__global__ void __launch_bounds__(kWeightThreads) cache4_weight_again_kernel(const Cache4 c, const Cache4Attention a, const Rows rows, const int row_blocks) {
  using R = Record<D>;
  constexpr int kTile = tile_tokens(D);
  griddep_launch_dependents();
  fence_ahead();
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  long long none;
  const long long total = all_units(c, a.counts, 0, 0, &none) * c.H;
  const Shares shares(total, gridDim.x * kWeightWarps);
  const int worker = shares.here();
  const bool used = worker < shares.workers;
  Cursor k;
  if (used) k = cursor_at(c, a.counts, c.H, 0, shares.begin(worker), shares.begin(worker + 1));
  griddep_wait();          // lengths were there before the first kernel started
  if (!used) return;       // behind the wait: this grid's end has to be behind that of the ones in front
  const int mask = (1 << c.page_shift) - 1;
  while (k.t < k.end) {
    const int run = k.end - k.t;
    for (int block = 0; block < row_blocks; ++block) {
      Query<D, NT> f;
      load_query<D, NT, kBf16>(f, c, a, rows, k.b, k.item, 8 * NT * block, k.n);
      float lse[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = 8 * (NT * block + nt) + 2 * q4 + i, t = row / rows.group, hq = k.item * rows.group + row - t * rows.group;
          if (row >= rows.count) f.last[nt][i] = -1;
          lse[nt][i] = f.last[nt][i] >= 0 ? a.lse[(static_cast<int64_t>(k.b) * a.Hq + hq) * a.S + t] * kLog2e : 0.f;
        }
      for (int t = kTile / 16 * k.t; t < kTile / 16 * (k.t + run); ++t) {
        const int slot = 16 * t;
        int64_t page;
        if (slot >= k.n || !find_page(c, k.b, slot, &page)) continue;
        float s[NT][4];
        block_scores<D, NT, kBf16>(s, c.kv + page * c.kv_stride[0] + k.item * c.kv_stride[1] + static_cast<int64_t>(slot & mask) * R::kBytes, f);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (slot + g + 8 * (j >> 1) <= f.last[nt][j & 1]) sum[j >> 1] += ex2(fmaf(s[nt][j], f.factor[nt][j & 1], -lse[nt][j & 1]));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
          sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
          if (q4 == 0 && slot + g + 8 * i < k.n)
            c.weight[page * c.weight_stride[0] + k.item * c.weight_stride[1] + (slot & mask) + g + 8 * i] += sum[i];
        }
      }
    }
    next_item(k, c, a.counts, c.H, 0);
  }
}

// Sixteen query rows at a time where there are more than eight: the cache is read half as often.  At D = 256 the
// accumulators of sixteen rows leave no room for anything else.
bool sixteen_rows(int D, int rows) { return D <= 128 && rows > 8; }

// Bytes of the scores of the longest sequences that the table allows.
size_t score_bytes(const Cache4& c, int rows) {
  const size_t tiles = static_cast<size_t>(c.B) * c.H * (((static_cast<size_t>(c.max_pages) << c.page_shift) + tile_tokens(c.D) - 1) / tile_tokens(c.D));
  return tiles * rows * tile_tokens(c.D) * sizeof(float);
}
// The scores are kept for the weights where a token's fit beside its record: one block of rows, and no more than half
// of what the cache itself takes.  They are placed by slot, so what counts is how long the table lets sequences be, which may be far
// more than there are pages: 2 sequences of 131072 tokens, 64 heads over 8, bf16, with a table that fits and one four times as
// wide, 109 and 181 us (D = 128), 76 and 130 (D = 64).  Four sequences of 32768 tokens, 8 heads, fp16, kept against computed
// again, us: D = 128, 8 / 16 rows, 65 / 99 against 102 / 127; D = 64, 8 rows, 47 against 73 (16 are always computed again, 87);
// D = 256, 8 rows, 98 against 146.
bool keeps_scores(const Cache4& c, int Hq, int S) {
  const int rows = Hq / c.H * S, block = sixteen_rows(c.D, rows) ? 16 : 8;
  const size_t cache_bytes = (static_cast<size_t>(c.pages) << c.page_shift) * c.H * (c.D * 5 / 4);
  return c.weight != nullptr && rows <= block && score_bytes(c, rows) <= cache_bytes / 2;
}

template <int D, int NT, bool kBf16>
cudaError_t launch_one(const Cache4& c, const Cache4Attention& a, int sm_count, cudaStream_t stream, long long* launches) {
  Rows rows;
  rows.group = a.Hq / c.H;
  rows.count = rows.group * a.S;
  const int row_blocks = (rows.count + 8 * NT - 1) / (8 * NT);
  using Sh = Shape<D, NT>;
  const int grid = sm_count;
  const bool pdl = option_pdl() != 0, keep = keeps_scores(c, a.Hq, a.S);
  static std::atomic<unsigned long long> smem_done{0};   // per kernel instantiation, bit per device
  cudaError_t e = set_dynamic_smem_once(smem_done, reinterpret_cast<const void*>(cache4_attention_kernel<D, NT, kBf16>), Sh::kRingBytes);
  if (e != cudaSuccess) return e;
  e = launch_persistent(cache4_attention_kernel<D, NT, kBf16>, grid, Sh::kThreads, Sh::kRingBytes, stream, pdl, c, a, rows, row_blocks, keep, option_wait_limit_ns(),
                        option_test_drop_load());
  if (e != cudaSuccess) return e;
  *launches += 1;
  // Where items are cut into many pieces, every row gets a CTA of its own, with a warp for every eight pieces.
  const int items = c.B * c.H * row_blocks;
  const long long pieces = static_cast<long long>(grid) * Sh::kWarps / items;
  const bool many_pieces = pieces > 8;
  const int rows_each = many_pieces ? 1 : 8 * NT;
  int join_threads = kJoinThreads;
  while (join_threads < kJoinMost && many_pieces && pieces > join_threads / 4) join_threads *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items), static_cast<unsigned>(many_pieces ? (rows.count < 8 * NT ? rows.count : 8 * NT) : 1));
  cfg.blockDim = dim3(join_threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, cache4_join_kernel<D, NT, kBf16>, c, a, rows, row_blocks, grid * Sh::kWarps, rows_each);
  if (e != cudaSuccess) return e;
  *launches += 1;
  if (c.weight != nullptr) {
    if (keep)
      e = launch_persistent(cache4_weight_kernel<tile_tokens(D)>, 8 * sm_count, kWeightThreads, 0, stream, pdl, c, a, rows);
    else
      e = launch_persistent(cache4_weight_again_kernel<D, NT, kBf16>, 4 * sm_count, kWeightThreads, 0, stream, pdl, c, a, rows, row_blocks);
    if (e == cudaSuccess) *launches += 1;
  }
  return e;
}

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
  return static_cast<size_t>(sm_count) * Shape<D, NT>::kWarps * 2 * piece_floats<D, NT>() * sizeof(float);
}
// The pieces, then the kept scores.
Cache4Workspace cache4_attention_workspace(const Cache4& c, int Hq, int S, int sm_count) {
  const int rows = Hq / c.H * S;
  const bool wide = sixteen_rows(c.D, rows);
  Cache4Workspace w;
  w.pieces = c.D == 64    ? (wide ? pieces_bytes<64, 2>(sm_count) : pieces_bytes<64, 1>(sm_count))
             : c.D == 128 ? (wide ? pieces_bytes<128, 2>(sm_count) : pieces_bytes<128, 1>(sm_count))
                          : pieces_bytes<256, 1>(sm_count);
  w.total = w.pieces + (keeps_scores(c, Hq, S) ? score_bytes(c, rows) : 0);
  return w;
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
