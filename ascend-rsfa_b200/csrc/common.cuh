// Types shared by the kernels and the C-ABI dispatcher.
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

namespace rsfa {

// One attention problem as the kernels see it: raw pointers plus element strides.
struct FwdParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;  // may be null
  int B, H, S, D;
  int64_t q_stride[3];  // batch, head, row (the innermost stride is 1)
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t o_stride[3];
  int causal;
  float sm_scale;
  int bf16;
  int tile_n;   // keys per tile on the tcgen05 path: 128 (single-buffered S) or 64 (double-buffered S)
  int variant;  // the "tcgen05_variant" option: -1 automatic, 0 / 1 / 2 force a kernel of the family
  int* status;                 // device status word, never null
  // Work queue of the persistent kernels: word [0] hands out work items, word [1] counts the CTAs
  // that have finished.  Both are zero before a launch; the CTA that finishes last puts them back
  // to zero, so the next launch that gets this pair needs no memset in front of it.
  unsigned int* tile_counter;
  unsigned long long wait_limit_ns;
  int pdl;             // 1: launch with programmatic stream serialisation (the "pdl" option)
  // Test hook (the "test_drop_load" option, -1 = off): the producer of the 128-key tcgen05 kernel
  // leaves out its n-th K/V tile load together with the barrier arrival that announces it, and the
  // kernel for a single key tile those of the heads from n on among the loads it starts with.  Nothing
  // is in flight for that tile and no address is touched; the consumer's bounded wait simply runs
  // out, which is how the tests reach the wait-expired path on a healthy GPU.
  int test_drop_load;
#ifdef RSFA_TRACE
  unsigned long long* trace;  // debug builds only: per-role event log of CTA 0
#endif
};

// A paged cache of 4-bit records (see rsfa_cache4 in rsfa.h) as the kernels see it.
struct Cache4 {
  uint8_t* kv;
  float* weight;        // may be null
  int* position;        // may be null
  const int* table;     // [B][max_pages] page of every page_size slots
  const int* lengths;   // [B]
  int64_t kv_stride[2];        // bytes: page, head
  int64_t weight_stride[2];    // elements: page, head
  int64_t position_stride[2];
  int64_t table_stride;        // elements: sequence
  int B, H, D, pages, max_pages;
  int page_shift;              // page_size = 1 << page_shift
  int bf16;
  int* status;                 // device status word, never null
};

struct RotaryParams {
  const void* x[2];        // q and k; k may be absent (heads[1] = 0)
  void* y[2];
  int64_t x_stride[2][3];  // batch, head, row
  int64_t y_stride[2][3];
  int heads[2];
  const float* table;      // [table_length][R / 2][2]: cosine and sine
  const void* positions;   // may be null: 0 .. S - 1
  int positions_64;        // int64 instead of int32
  int64_t pos_stride[2];   // batch, row
  int B, S, D, R, table_length;
  int interleaved, inverse, bf16;
  int* status;
};

struct Cache4Rows {        // dense K and V rows that go into or come out of a cache
  void* k;
  void* v;
  int64_t k_stride[3];     // batch, head, row
  int64_t v_stride[3];
  int S;
  const int* counts;       // append: rows of each sequence that count; may be null: all
  const int* starts;       // read: first slot of each sequence; may be null: 0
  const int* positions;    // append: may be null
  int64_t positions_stride[2];
};

struct Cache4Attention {
  const void* q;
  void* o;
  float* lse;              // may be null
  int64_t q_stride[3], o_stride[3];
  int Hq, S;
  const int* counts;       // may be null
  float sm_scale;
  float* pieces;           // workspace: partial sums
  float* scores;           // workspace: scores kept for the weights
};

struct Cache4Evict {
  int budget, recent;
  int most_moves;          // of a head; what `moves` has room for
  int* new_lengths;
  int* moves;              // workspace
};

// What a call needs of the current device: multiprocessors and the status word.  begin_call refuses under the
// "check_status" option as rsfa_fwd does; end_call turns a launch's outcome into a return code.
struct CallScratch {
  int sm_count;
  int* status;
  int* status_mirror;
};
int begin_call(CallScratch* out);
int end_call(const CallScratch& d, cudaStream_t stream, cudaError_t e, long long launches);

// Raises a kernel's dynamic shared-memory limit once per device instead of on every call (the
// attribute stays with the function in that device's context).  `done` is a bit mask by device
// ordinal, one per kernel instantiation (a static of the launcher that owns the kernel).
inline cudaError_t set_dynamic_smem_once(std::atomic<unsigned long long>& done, const void* kern, int bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && ((done.load(std::memory_order_acquire) >> dev) & 1ull)) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  return e;
}

// Launchers implemented in the kernel translation units.  Each returns a cudaError_t
// from the launch itself and bumps *launches by the number of kernels it started.
cudaError_t launch_fwd_generic(const FwdParams& p, cudaStream_t stream, long long* launches);
// CTAs the short-sequence kernel launches: one per (batch, head, block of 64 query rows), all on grid.x.
long long generic_grid_blocks(int B, int H, int S);
cudaError_t launch_fwd_tcgen05(const FwdParams& p, int sm_count, cudaStream_t stream,
                               long long* launches);
// The single-key-tile kernel (fwd_short.cu), S <= 128 at D <= 64 and S <= 64 at D = 128.
cudaError_t launch_fwd_short(const FwdParams& p, int sm_count, cudaStream_t stream, long long* launches);
bool short_fits(int S, int D, float sm_scale);
// The double-buffered-S family (D = 64, 128, 256), selected by launch_fwd_tcgen05.
cudaError_t launch_fwd_tcgen05_db(const FwdParams& p, int sm_count, cudaStream_t stream,
                                  long long* launches);
// Its form for D <= 64 with one Q tile per CTA, and whether a launch is better off with it.
cudaError_t launch_fwd_tcgen05_db_single(const FwdParams& p, int sm_count, cudaStream_t stream, long long* launches);
bool single_tiles_pay(const FwdParams& p, int sm_count);
// The D = 64 kernel with P in tensor-memory columns of its own (fwd_tcgen05_sp.cu), selected by launch_fwd_tcgen05.
cudaError_t launch_fwd_tcgen05_sp(const FwdParams& p, int sm_count, cudaStream_t stream, long long* launches);
// Whether a problem's work items can be numbered in that kernel's scheduler ring (fewer than 2^27).
bool tcgen05_sp_fits(const FwdParams& p);
// Tile the tcgen05 family runs for a problem: the requested (block_m, block_n) when that tile is
// instantiated for D, otherwise the tile table's row for (S, D, causal).  `variant` = -1 lets the
// request / table decide, 0 forces 128-key tiles with single-buffered S, 1 forces 64-key tiles (D <= 128
// only), 2 forces 128-key tiles with the separate-P kernel where it exists (D = 64).
void tcgen05_resolve_tile(int S, int D, int causal, int req_bm, int req_bn, int variant, int* bm, int* bn);
// The operators around attention (rotary.cu, cache4_rows.cu, cache4_attention.cu, cache4_evict.cu).
cudaError_t launch_rotary(const RotaryParams& p, int sm_count, cudaStream_t stream, long long* launches);
cudaError_t launch_rotary_table(float* table, int length, int dim, const double* freq_args, int scaling, cudaStream_t stream,
                                long long* launches);
cudaError_t launch_cache4_append(const Cache4& c, const Cache4Rows& r, cudaStream_t stream, long long* launches);
cudaError_t launch_cache4_read(const Cache4& c, const Cache4Rows& r, cudaStream_t stream, long long* launches);
cudaError_t launch_cache4_attention(const Cache4& c, const Cache4Attention& a, int sm_count, cudaStream_t stream, long long* launches);
struct Cache4Workspace {
  size_t pieces, total;   // bytes
};
Cache4Workspace cache4_attention_workspace(const Cache4& c, int Hq, int S, int sm_count);
cudaError_t launch_cache4_evict(const Cache4& c, const Cache4Evict& e, int sm_count, cudaStream_t stream, long long* launches);
int cache4_most_moves(const Cache4& c, int budget);
size_t cache4_evict_workspace(int B, int H, int most_moves);
// Adds to the process-wide kernel-launch counter behind rsfa_launch_count().
void count_launches(long long n);
// Current values of the "wait_limit_ms" (in ns), "pdl" and "test_drop_load" options.
unsigned long long option_wait_limit_ns();
int option_pdl();
int option_test_drop_load();
// Device address of the status word in the static scratch block of rsfa_fwd_noalloc on `device`, or
// null while that entry point has not been used there.
int* noalloc_status_word(int device);
// True when the tcgen05 kernel is instantiated for this head dimension.
bool tcgen05_supports(int S, int D, float sm_scale);

}  // namespace rsfa
