// Eviction from a paged cache of 4-bit records by accumulated attention weight.
//
// Of the n tokens of a sequence, every K/V head keeps `budget`: those whose position is among the newest `recent`
// ones (position > newest - recent), then those with the largest weight, the lowest slot first among equals.  The
// kept tokens beyond slot `budget` move into the slots below it that are given up, both in rising order, so nothing
// else moves and the order of the others stays; attention does not depend on the order.
//
// Two launches.  select: one CTA per (sequence, head) finds the budget-th largest key with three histograms of 11,
// 11 and 10 bits (a weight is not negative, so its bits order as an integer; a protected token has the largest key) and
// lists the moves by prefix sums over the slots.  move: the listed records, spread over the whole device.
// What bounds it: the latency of the passes over n keys of one CTA and, where heads are fewer than multiprocessors, that one
// CTA's shared memory; the traffic, 8 bytes per token and 2 * 5 D / 4 per move, is small next to a step's attention.
// 256 heads of 2049 slots: select 12.9 us, one move each 3.9 us.  32 heads of 16384 slots cut to a quarter: select 18.6 us,
// move 4.5 us.
#include "../../include/rsfa.h"
#include "ops_common.cuh"

namespace rsfa {
namespace {

constexpr int kSlotsEach = 4;              // neighbouring slots of a thread: one page, one address, one access of shared memory
constexpr int kBins = 2048;
constexpr int kKeysInShared = 20 * 1024;   // slots whose keys and positions are kept in shared memory; of longer sequences
                                           // the others are read again in every pass
constexpr int kPagesInShared = 2048;       // and page numbers
constexpr int kSelectBytes = kKeysInShared * 8 + kPagesInShared * 4;
constexpr int kMoveThreads = 256;
constexpr uint32_t kProtected = 0xffffffffu;

__device__ __forceinline__ int64_t moves_at(const Cache4Evict& e, int bh) { return static_cast<int64_t>(bh) * (2ll * e.most_moves + 2); }

// Exclusive prefix sum over the block and the block's total.
template <int kWarps>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t sum = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += u;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  const uint32_t w = lane < kWarps ? warp_sums[lane] : 0u;
  uint32_t ws = w;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, ws, d);
    if (lane >= d) ws += u;
  }
  *total = __shfl_sync(0xffffffffu, ws, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, ws - w, warp);
  __syncthreads();                              // warp_sums may be written again
  return before + sum - v;
}

template <int kSelectThreads>
__global__ void __launch_bounds__(kSelectThreads) cache4_select_kernel(const Cache4 c, const Cache4Evict e) {
  extern __shared__ __align__(16) uint32_t kept_slots[];    // keys, then positions of the first `in_shared` slots, then page numbers
  __shared__ uint32_t hist[kBins];
  constexpr int kSelectWarps = kSelectThreads / 32;
  __shared__ uint32_t warp_sums[kSelectWarps];
  __shared__ int newest_word;
  __shared__ uint32_t found_bin, found_above;
  griddep_launch_dependents();
  griddep_wait();
  const int bh = blockIdx.x, b = bh / c.H, h = bh - b * c.H;
  const int tid = threadIdx.x;
  const int n = tokens_of(c, b);
  int* count = e.moves + moves_at(e, bh);
  int2* moves = reinterpret_cast<int2*>(count + 2);
  if (tid == 0 && h == 0) e.new_lengths[b] = min(n, e.budget);
  if (n <= e.budget) {
    if (tid == 0) *count = 0;
    return;
  }
  const int mask = (1 << c.page_shift) - 1;
  // slots are taken in fours; what stands behind the last one has key 0, which no real key is below
  const int n4 = (n + 3) & ~3, in_shared = min(n4, kKeysInShared), pages_in_shared = min((n + mask) >> c.page_shift, kPagesInShared);
  uint32_t* const keys = kept_slots;
  int* const positions = reinterpret_cast<int*>(kept_slots + in_shared);
  int* const page_ids = positions + in_shared;
  if (tid == 0) newest_word = INT_MIN;
  for (int i = tid; i < pages_in_shared; i += kSelectThreads) {
    int64_t page;
    page_ids[i] = find_page(c, b, i << c.page_shift, &page) ? static_cast<int>(page) : -1;
  }
  __syncthreads();
  auto page_of = [&](int slot) -> int64_t {
    if ((slot >> c.page_shift) < pages_in_shared) return page_ids[slot >> c.page_shift];
    int64_t page;
    return find_page(c, b, slot, &page) ? page : -1;
  };
  // positions and weight bits of four slots; those without a page, or behind the last one, are the oldest and lightest
  auto read_slots = [&](int slot, int4* position, uint4* weight) {
    const int64_t page = page_of(slot);
    int p[4] = {INT_MIN, INT_MIN, INT_MIN, INT_MIN};
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (page >= 0) {
      const int* pp = c.position + page * c.position_stride[0] + h * c.position_stride[1] + (slot & mask);
      const float* wp = c.weight + page * c.weight_stride[0] + h * c.weight_stride[1] + (slot & mask);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = wp[j];
        const int q = pp[j];
        if (slot + j < n) {
          w[j] = f > 0.f ? __float_as_uint(f) : 0u;                // NaN, negative: as no weight
          p[j] = q;
        }
      }
    }
    *position = make_int4(p[0], p[1], p[2], p[3]);
    *weight = make_uint4(w[0], w[1], w[2], w[3]);
  };
  int newest = INT_MIN;
#pragma unroll 2
  for (int i = 4 * tid; i < n; i += 4 * kSelectThreads) {
    int4 p;
    uint4 w;
    read_slots(i, &p, &w);
    newest = max(max(newest, max(p.x, p.y)), max(p.z, p.w));
    if (i < in_shared) {
      *reinterpret_cast<uint4*>(keys + i) = w;
      *reinterpret_cast<int4*>(positions + i) = p;
    }
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if ((tid & 31) == 0) atomicMax(&newest_word, newest);
  __syncthreads();
  // the largest position that is not protected, within what 32 bits hold
  const int oldest_kept = static_cast<int>(max(static_cast<long long>(newest_word) - e.recent, static_cast<long long>(INT_MIN)));
  auto protect = [&](const int4& p, uint4 w) {
    if (p.x > oldest_kept) w.x = kProtected;
    if (p.y > oldest_kept) w.y = kProtected;
    if (p.z > oldest_kept) w.z = kProtected;
    if (p.w > oldest_kept) w.w = kProtected;
    return w;
  };
  for (int i = 4 * tid; i < in_shared; i += 4 * kSelectThreads) {  // each thread's own slots
    uint4* k = reinterpret_cast<uint4*>(keys + i);
    *k = protect(*reinterpret_cast<const int4*>(positions + i), *k);
  }
  auto keys_at = [&](int slot) -> uint4 {
    if (slot < in_shared) return *reinterpret_cast<const uint4*>(keys + slot);
    int4 p;
    uint4 w;
    read_slots(slot, &p, &w);
    return protect(p, w);
  };

  // ---- the budget-th largest key, by digits from the top
  uint32_t prefix = 0, want = e.budget;         // `want` keys are to come from those that share the prefix
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit_mask = pass == 2 ? 1023u : 2047u;
    const uint32_t above = pass == 0 ? 0u : pass == 1 ? ~0u << 21 : ~0u << 10;
    for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
#pragma unroll 2
    for (int i = 4 * tid; i < n; i += 4 * kSelectThreads) {
      const uint4 four = keys_at(i);
      const uint32_t key[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (((key[j] ^ prefix) & above) == 0) atomicAdd(&hist[(key[j] >> shift) & digit_mask], 1u);
    }
    __syncthreads();
    // neighbouring bins of a thread, from the highest down
    constexpr int kEach = kBins / kSelectThreads;
    const int hi = kBins - 1 - kEach * tid;
    uint32_t mine = 0, total;
#pragma unroll
    for (int j = 0; j < kEach; ++j) mine += hist[hi - j];
    uint32_t before = block_scan<kSelectWarps>(mine, warp_sums, &total);
    if (before < want && want <= before + mine) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const uint32_t in_bin = hist[hi - j];
        if (before < want && want <= before + in_bin) {
          found_bin = hi - j;
          found_above = before;
        }
        before += in_bin;
      }
    }
    __syncthreads();
    prefix |= found_bin << shift;
    want -= found_above;
  }

  // ---- kept: larger keys, and the first `want` slots of equal ones; the moves in rising order
  uint32_t equals = 0, holes = 0, movers = 0;
  for (int base = 0; base < n; base += kSelectThreads * kSlotsEach) {
    const int first = base + tid * kSlotsEach;
    const uint4 four = first < n ? keys_at(first) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t key[kSlotsEach] = {four.x, four.y, four.z, four.w};
    uint32_t eq = 0;
#pragma unroll
    for (int j = 0; j < kSlotsEach; ++j) eq += first + j < n && key[j] == prefix;
    uint32_t total;
    uint32_t rank = equals + block_scan<kSelectWarps>(eq, warp_sums, &total);
    equals += total;
    uint32_t is_hole = 0, is_mover = 0;
#pragma unroll
    for (int j = 0; j < kSlotsEach; ++j) {
      const int slot = first + j;
      if (slot < n) {
        const bool same = key[j] == prefix;
        const bool kept = key[j] > prefix || (same && rank < want);
        rank += same;
        if (slot < e.budget && !kept) is_hole |= 1u << j;
        if (slot >= e.budget && kept) is_mover |= 1u << j;
      }
    }
    // both counts of a round's slots, 4096 at most, in one word
    const uint32_t at = block_scan<kSelectWarps>(__popc(is_hole) | (__popc(is_mover) << 16), warp_sums, &total);
    uint32_t hole_at = holes + (at & 0xffffu), mover_at = movers + (at >> 16);
#pragma unroll
    for (int j = 0; j < kSlotsEach; ++j) {
      if (is_hole >> j & 1) moves[hole_at++].x = first + j;
      if (is_mover >> j & 1) moves[mover_at++].y = first + j;
    }
    holes += total & 0xffffu;
    movers += total >> 16;
  }
  if (tid == 0) *count = static_cast<int>(holes);   // as many as movers: budget slots are kept
}

// Pieces of 16 bytes, and one more per record for its weight and position.
__global__ void __launch_bounds__(kMoveThreads) cache4_move_kernel(const Cache4 c, const Cache4Evict e, const int pieces) {
  griddep_launch_dependents();
  griddep_wait();
  const int bh = blockIdx.x, b = bh / c.H, h = bh - b * c.H;
  const int* count = e.moves + moves_at(e, bh);
  const int2* moves = reinterpret_cast<const int2*>(count + 2);
  const long long total = static_cast<long long>(*count) * pieces;
  const int mask = (1 << c.page_shift) - 1;
  for (long long i = static_cast<long long>(blockIdx.y) * kMoveThreads + threadIdx.x; i < total; i += static_cast<long long>(gridDim.y) * kMoveThreads) {
    const int m = static_cast<int>(i / pieces), piece = static_cast<int>(i - static_cast<long long>(m) * pieces);
    const int2 move = moves[m];                 // to, from
    int64_t to, from;
    if (!find_page(c, b, move.x, &to) || !find_page(c, b, move.y, &from)) continue;
    if (piece < pieces - 1) {
      const int64_t rec = 16ll * (pieces - 1);
      const uint8_t* src = c.kv + from * c.kv_stride[0] + h * c.kv_stride[1] + (move.y & mask) * rec + 16 * piece;
      uint8_t* dst = c.kv + to * c.kv_stride[0] + h * c.kv_stride[1] + (move.x & mask) * rec + 16 * piece;
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
    } else {
      c.weight[to * c.weight_stride[0] + h * c.weight_stride[1] + (move.x & mask)] =
          c.weight[from * c.weight_stride[0] + h * c.weight_stride[1] + (move.y & mask)];
      c.position[to * c.position_stride[0] + h * c.position_stride[1] + (move.x & mask)] =
          c.position[from * c.position_stride[0] + h * c.position_stride[1] + (move.y & mask)];
    }
  }
}

}  // namespace

// A record moves from a slot beyond the budget to one within it: no more of them than there are of either.
int cache4_most_moves(const Cache4& c, int budget) {
  const int room = c.max_pages << c.page_shift;
  return room <= budget ? 0 : room - budget < budget ? room - budget : budget;
}
size_t cache4_evict_workspace(int B, int H, int most_moves) {
  return static_cast<size_t>(B) * H * (2ull * most_moves + 2) * sizeof(int);
}

cudaError_t launch_cache4_evict(const Cache4& c, const Cache4Evict& ev, int sm_count, cudaStream_t stream, long long* launches) {
  const long long room = static_cast<long long>(c.max_pages) << c.page_shift;
  const int smem = static_cast<int>(room < kKeysInShared ? room : kKeysInShared) * 8 + (c.max_pages < kPagesInShared ? c.max_pages : kPagesInShared) * 4;
  const int heads = c.B * c.H;
  cudaError_t e;
  // Short sequences with 256 threads, of which every multiprocessor holds several CTAs: 256 heads of 2049 slots
  // 15.5 -> 13.0 us of select alone.  (By what the table allows, as the lengths are on the device; with the move behind it, which
  // starts while select ends, a call takes 17.7 us with a table that fits and 17.0 with one of 131072 slots.)
  if (room <= 4096) {
    e = launch_persistent(cache4_select_kernel<256>, heads, 256, smem, stream, option_pdl() != 0, c, ev);
  } else {
    static std::atomic<unsigned long long> smem_done{0};
    e = set_dynamic_smem_once(smem_done, reinterpret_cast<const void*>(cache4_select_kernel<1024>), kSelectBytes);
    if (e != cudaSuccess) return e;
    e = launch_persistent(cache4_select_kernel<1024>, heads, 1024, smem, stream, option_pdl() != 0, c, ev);
  }
  if (e != cudaSuccess) return e;
  *launches += 1;
  const int pieces = c.D * 5 / 4 / 16 + 1;
  // enough CTAs for a large cut, and no more than its moves could keep busy
  long long each = (8ll * sm_count + heads - 1) / heads;
  const long long most = (static_cast<long long>(ev.most_moves) * pieces + kMoveThreads - 1) / kMoveThreads;
  if (each > most) each = most;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(heads), static_cast<unsigned>(each < 1 ? 1 : each));
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option_pdl() ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, cache4_move_kernel, c, ev, pieces);
  if (e == cudaSuccess) *launches += 1;
  return e;
}

}  // namespace rsfa
