/*
 * rsfa.h — C ABI of the B200 FlashAttention-2 forward library (librsfa_b200.so).
 *
 * The library is the device side of the Python operator
 *   ascend_rsfa.flash_attention_forward.attention(q, k, v, causal, sm_scale, BLOCK_M, BLOCK_N)
 * and of get_tiling(batch, heads, seq, head_dim, causal).  All tensors are
 * [B, H, S, D] with 16-bit elements; all pointers are plain device (or, where
 * stated, host) addresses; sizes are ints; nothing here depends on PyTorch.
 * Every function returns RSFA_OK (0) or a negative RSFA_ERR_* code and never
 * aborts the process.  rsfa_strerror() names a code.
 *
 * Citations of the form file:line point into the reference project
 * (ascend_rsfa/flash_attention_forward.py unless another file is named).
 */
#ifndef RSFA_H_
#define RSFA_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define RSFA_API __attribute__((visibility("default")))
#else
#define RSFA_API
#endif

#define RSFA_OK 0
#define RSFA_ERR_INVALID_ARGUMENT (-1) /* bad shape, stride, alignment, tile or dtype           */
#define RSFA_ERR_UNSUPPORTED (-2)      /* legal for the reference, not built here               */
#define RSFA_ERR_CUDA (-3)             /* a CUDA runtime / driver call failed                   */
#define RSFA_ERR_DEVICE_STATUS (-4)    /* a kernel reported a non-zero status (bounded wait...) */
#define RSFA_ERR_NO_DEVICE (-5)        /* no CUDA device, or not an sm_100 device               */
#define RSFA_ERR_TOO_LARGE (-6)        /* beyond rsfa_fwd_noalloc's fixed scratch, or > 2^31-1 CTAs */

#define RSFA_DTYPE_F16 0
#define RSFA_DTYPE_BF16 1

/* Kernel families a call can be routed to (see rsfa_select_path). */
#define RSFA_PATH_GENERIC 0 /* mma.sync kernel: any S, D in {16,32,64,128,256}; the smallest tiles, scale <= 0 */
#define RSFA_PATH_TCGEN05 1 /* warp-specialised tcgen05 / TMEM / TMA kernel                         */
/*
 * Sequences of one key tile - S <= 128 at D <= 64, S <= 64 at D = 128, sm_scale > 0 - run on a kernel of
 * their own (TMA-fed, warp-level MMA, csrc/fwd_short.cu) whichever of the two families their size belongs
 * to, unless "force_path" or "tcgen05_variant" asks for a particular kernel.  rsfa_select_path,
 * rsfa_get_tiling and rsfa_work_items name the family and its tile and count of items by size alone.
 */

/*
 * Forward attention on device tensors.  Replaces _attention.forward (:547-616)
 * with everything it dispatches to: _attn_fwd_small / _attn_fwd_small_causal
 * (:26-159), _attn_fwd with _attn_fwd_inner / _attn_fwd_inner_d64_nc (:163-404)
 * and the two-launch causal split _run_causal_split (:493-541).
 *
 *   q, k, v, o   device pointers, element (b,h,s,d) at base + b*st[0] + h*st[1] + s*st[2] + d*st[3]
 *   lse          optional device pointer to B*H*S floats (contiguous): m + log(l) per row in
 *                natural-log units (:400-404); may be NULL.  Written for causal calls too.
 *   strides      16 element strides: q[4], k[4], v[4], o[4].  The innermost stride must be 1, the
 *                others multiples of 8 elements, and the base pointers 16-byte aligned.
 *   causal       0/1; the mask keeps key j <= query i, square and aligned top-left (:153, :194).
 *   sm_scale     multiplies q.k before the softmax (:84, :199).
 *   block_m/n    the reference's BLOCK_M / BLOCK_N.  Results do not depend on them; they are a
 *                request that is honoured when such a tile is instantiated and otherwise replaced
 *                by the table's choice (rsfa_get_tiling).  Must be positive.  Launches too small to
 *                fill the device, sequences of one key tile and, at D <= 64, short and medium sequences
 *                run on forms of the kernels made for them whatever was asked for.
 *   dtype        RSFA_DTYPE_F16 or RSFA_DTYPE_BF16 (:698 tests one bf16 case).
 *   stream       a cudaStream_t (NULL = default stream).  The call is asynchronous like the
 *                reference's kernel launches; it does not synchronise.
 *
 * Concurrency: calls on different streams of one device may overlap on the GPU.  Every call is one
 * kernel launch and takes a work queue of its own out of 1024 per device (the kernel puts it back to
 * zero when it ends); nothing else in device memory is shared between calls except the status word,
 * which is per device.
 *
 * Errors: D outside {16,32,64,128,256} or mismatched (the reference asserts, :551-554), B/H/S < 1,
 * misaligned pointers or strides -> RSFA_ERR_INVALID_ARGUMENT.  A device status left by an earlier
 * launch on the same device is reported by rsfa_device_status, not here.
 */
RSFA_API int rsfa_fwd(const void* q, const void* k, const void* v, void* o, float* lse,
             int B, int H, int S, int D, const int64_t* strides,
             int causal, float sm_scale, int block_m, int block_n, int dtype, void* stream);

/*
 * The same operator on HOST buffers (contiguous [B,H,S,D]); the library stages heads through the
 * device in slabs, overlapping host->device copies, kernels and device->host copies on its own
 * streams, and returns when o_host (and lse_host, if not NULL) is complete.  This is the call the
 * reference's harness makes when its tensors start on the host: tensor creation + attention() +
 * synchronize (benchmarks/run_final_benchmark.py:104-124).  Buffers may be pageable; pinned
 * buffers copy faster.  `device` is the CUDA ordinal to use.  Calls for one device share its staging
 * buffers and streams: issue them one at a time per device (different devices are independent).
 */
RSFA_API int rsfa_fwd_host(const void* q_host, const void* k_host, const void* v_host, void* o_host,
                  float* lse_host, int B, int H, int S, int D, int causal, float sm_scale,
                  int block_m, int block_n, int dtype, int device);

/*
 * rsfa_fwd for callers that must not allocate device memory.  It has no counterpart in the
 * reference; it exists for hosts where a cudaMalloc inside an operator call is not acceptable:
 * servers that give all device memory to their own arena at start-up, latency-critical loops in
 * which an allocation may stall the device, plugins whose memory is accounted by the embedding
 * process.  rsfa_fwd keeps its work-queue counter and status word in a buffer it cudaMallocs on
 * first use; this entry point runs the same tcgen05 kernel with that scratch in a 256-byte block
 * of static device memory inside the library (held by every GPU that loads the library until the
 * process exits) and calls no cudaMalloc, cudaFree or other allocating routine.
 *
 * Arguments as rsfa_fwd, without block_m / block_n: the tile table decides, so either tcgen05
 * kernel family may run, as in rsfa_fwd (64-key tiles at D = 256 and for short causal sequences,
 * 128-key tiles otherwise, the separate-P kernel at D <= 64).
 * Every in-kernel wait is bounded by the "wait_limit_ms" option, as in rsfa_fwd.  Limits: only
 * shapes the tcgen05 kernels are built for (sm_scale > 0; D = 16 and 32 run on the D = 64 kernel) -> otherwise
 * RSFA_ERR_UNSUPPORTED; at most 2^30 work items (B * H * ceil(S / 256), or ceil(S / 128) at D = 256), because the queue counter
 * is a single 32-bit word of the block -> otherwise RSFA_ERR_TOO_LARGE.
 *
 * The first call on a device looks up the device address of the static block (one
 * cudaGetSymbolAddress with that device current); make that first call outside any stream
 * capture.  All calls on a device share the one block, which keeps the previous call's contents:
 * each call clears the work queue and the status word on `stream` before its kernel, so calls on
 * one stream are safe back to back, but two calls whose kernels can overlap on the GPU (different
 * streams, no dependency) race on the queue and must be ordered by the caller.  A bounded wait
 * that runs out leaves the output incomplete and a code in the block's status word, which
 * rsfa_device_status reports together with rsfa_fwd's (the next rsfa_fwd_noalloc call clears it).
 */
RSFA_API int rsfa_fwd_noalloc(const void* q, const void* k, const void* v, void* o, float* lse,
                              int B, int H, int S, int D, const int64_t* strides,
                              int causal, float sm_scale, int dtype, void* stream);

/*
 * ---------------------------------------------------------------------------------------------
 * Around attention: rotary positions, and a paged cache that holds K and V in 4 bits for decoding.
 * The reference has no counterpart.  All calls are asynchronous on `stream`, run on the current
 * device, allocate nothing (but the library's workspace on a device's first call, which therefore
 * is made outside stream capture) and keep nothing from one call for the next; scratch is the
 * caller's, and a scratch buffer belongs to one call at a time.  What lies in device memory cannot
 * be checked when a call is made: a kernel that finds a position, page number or length out of range
 * touches nothing outside, goes on (the results of that sequence have no meaning) and leaves
 * (2 << 16) | tag in the status word (rsfa_device_status): tag 1 a position outside the rotary table, 2 a
 * page outside the cache, 3 a length below zero or beyond the sequence's pages.
 */

/* How the angles of rotary positions are scaled for contexts longer than those of training. */
#define RSFA_ROTARY_NONE 0
#define RSFA_ROTARY_LINEAR 1 /* every angle divided by factor                                        */
#define RSFA_ROTARY_NTK 2    /* base times factor^(dim / (dim - 2)); dim = 2: as LINEAR               */
#define RSFA_ROTARY_YARN 3   /* a ramp over the pairs, from unscaled to divided by factor, between    */
                             /* those with high_turns and low_turns turns over original_length        */
#define RSFA_ROTARY_BANDS 4  /* the same between the two numbers of turns, linear in the turns        */

/*
 * The table of a rotation: table[p][i] = multiplier * (cos, sin)(p * f_i) for positions p < length and
 * pairs i < dim / 2, fp32, from angles in 64 bits; f_i = base^(-2 i / dim), scaled as asked for.
 * table: device, 16-byte aligned, length * dim floats; dim even, 2 ... 256; base > 1.  factor counts
 * unless scaling is NONE, original_length and the turns (0 < low_turns < high_turns) for YARN and BANDS.
 */
RSFA_API int rsfa_rotary_table(float* table, int length, int dim, double base, int scaling, double factor,
                               int original_length, double low_turns, double high_turns, double multiplier,
                               void* stream);

/*
 * Rotary positions on q [B,Hq,S,D] and k [B,Hk,S,D] in one launch (k and k_out NULL with Hk = 0: q alone).
 * The pair (a, b) of frequency i becomes (a c - b s, b c + a s), (c, s) = table[position][i]; pairs are
 * (i, i + rotary_dim / 2), or (2 i, 2 i + 1) if interleaved; dims from rotary_dim on are copied.  inverse: the
 * transposed rotation, which is the gradient.  strides: 16 element strides, q[4], k[4], q_out[4], k_out[4], as
 * rsfa_fwd asks for them; outputs do not overlap inputs.  rotary_dim: even, 2 ... D; multiples of 16 (8 if
 * interleaved) are fast.  positions: int32 (int64 if positions_64) with element strides (batch, row), 0 for
 * a row that all sequences share; NULL: 0 ... S - 1.  A row whose position is outside the table comes out as NaN.
 */
RSFA_API int rsfa_rotary(const void* q, const void* k, void* q_out, void* k_out, int B, int Hq, int Hk, int S, int D,
                         const int64_t* strides, const float* table, int table_length, int rotary_dim,
                         const void* positions, int positions_64, const int64_t* position_strides, int interleaved,
                         int inverse, int dtype, void* stream);

/*
 * A paged cache of 4-bit records.  Slot s of sequence b lies in page table[b * table_stride + s / page_size], row
 * s % page_size; lengths[b] slots are in use.  A record (one token of one K/V head) is 5 head_dim / 4 bytes:
 * head_dim / 2 of K codes, as many of V codes, then for K and for V a (scale, minimum) pair of `dtype` per group of
 * 32 dims; a value is scale * code + minimum.  The order of the codes is the kernels' own (csrc/ops_common.cuh).
 * head_dim 64, 128 or 256; page_size a power of two, 16 ... 1024; kv 16-byte aligned, its strides (bytes: page, head)
 * multiples of 16, a head's rows of a page contiguous; max_pages * page_size no more than 2^30.  weight (fp32) and
 * position (int32), one per record with element strides (page, head), are NULL where a call does not use them.
 * Sequences may share pages that a call only reads.
 */
typedef struct rsfa_cache4 {
  void* kv;
  float* weight;
  int* position;
  const int* table;
  const int* lengths;
  int64_t kv_stride[2];
  int64_t weight_stride[2];
  int64_t position_stride[2];
  int64_t table_stride;
  int batch, heads, head_dim, page_size, pages, max_pages, dtype;
} rsfa_cache4;

/*
 * K and V rows [B,heads,S,D] into the last slots of each sequence: row j < counts[b] (NULL: S) goes to slot
 * lengths[b] - counts[b] + j, so lengths is what they are WITH the new rows; slots below zero or behind the
 * pages are left out.  Per group the minimum, the scale 16-bit((max - min) / 15) and the nearest codes; a group
 * that holds an infinity or NaN reads back as NaN.  weight is set to 0 and position to positions[b][j] (element strides; given if position is).
 * strides: 8 element strides, k[4], v[4], as rsfa_fwd asks for them.
 */
RSFA_API int rsfa_cache4_append(const rsfa_cache4* cache, const void* k, const void* v, int S, const int64_t* strides,
                                const int* counts, const int* positions, const int64_t* position_strides, void* stream);

/* Slots starts[b] (NULL: 0) ... + N - 1 back to dense K and V rows [B,heads,N,D]; slots not in use are zero. */
RSFA_API int rsfa_cache4_read(const rsfa_cache4* cache, void* k, void* v, int N, const int64_t* strides,
                              const int* starts, void* stream);

/*
 * Attention of the last counts[b] (NULL: S) tokens of each sequence over its cache: query i of q [B,q_heads,S,D] sees the
 * slots up to lengths[b] - counts[b] + i, its own among them (append comes first).  q_heads is a multiple of heads;
 * K/V head h serves the query heads h * q_heads / heads ... .  o like q, both of cache->dtype; a row that sees nothing
 * (a sequence of length zero, a row of padding) is zero, its lse -infinity.  lse: [B,q_heads,S] fp32, natural log, may
 * be NULL unless cache->weight is given: weight[slot] then grows by the softmax weights that the token gets from all
 * query rows of its K/V head (and no page belongs to two sequences).  Results do not depend on timing.
 * strides: 8 element strides, q[4], o[4].
 * At most 2^40 tiles of 32 tokens for 8 query rows, counted by max_pages, else RSFA_ERR_TOO_LARGE.
 * workspace: rsfa_cache4_attention_workspace bytes (or a negative error), 16-byte aligned, no content asked for; with
 * weight it holds the scores, up to half the size of the cache.
 */
RSFA_API long long rsfa_cache4_attention_workspace(const rsfa_cache4* cache, int q_heads, int S);
RSFA_API int rsfa_cache4_attention(const rsfa_cache4* cache, const void* q, void* o, float* lse, int q_heads, int S,
                                   const int64_t* strides, const int* counts, float sm_scale, void* workspace,
                                   long long workspace_bytes, void* stream);

/*
 * Cuts every sequence back to `budget` slots, for each K/V head on its own: kept are the tokens at the newest `recent`
 * positions (position > largest - recent), then those of the largest weight, the lowest slot first among equals; a
 * weight that is negative or NaN counts as none.  Kept records beyond slot `budget` move, with weight and position, into
 * the slots below that are given up, both in rising order; nothing else is written.  new_lengths[b] =
 * min(lengths[b], budget), which is not lengths itself: other layers' caches may still need that.  0 <= recent <= budget.
 * No page may belong to two sequences.  workspace as above, for
 * most_moves = min(budget, max_pages * page_size - budget), 0 where that is negative: no more records of a head can move.
 */
RSFA_API long long rsfa_cache4_evict_workspace(int batch, int heads, int most_moves);
RSFA_API int rsfa_cache4_evict(const rsfa_cache4* cache, int budget, int recent, int* new_lengths, void* workspace,
                               long long workspace_bytes, void* stream);

/*
 * Tile lookup.  Replaces get_tiling (:624-665): the reference keys a 32-entry dict by the full
 * (Z, H, N_CTX, HEAD_DIM, causal) tuple and raises KeyError otherwise; here the table is keyed by
 * (S, D, causal) only, any B and H are accepted, and only tiles that are instantiated are returned.
 */
RSFA_API int rsfa_get_tiling(int B, int H, int S, int D, int causal, int* block_m, int* block_n);

/*
 * Which kernel family rsfa_fwd would use for this problem, and the tile it would run
 * (after snapping block_m/block_n).  Counterpart of the dispatch in _attention.forward (:564-610).
 * tile_m / tile_n may be NULL.  The answer goes by size alone: the tcgen05 family for every shape with
 * sm_scale > 0 except head dimension 16 at S <= 128 and sequences of at most 64 keys at D <= 64; which
 * form of a kernel, or the kernel for a single key tile, then runs is left open (see RSFA_PATH_*).
 */
RSFA_API int rsfa_select_path(int S, int D, int causal, float sm_scale, int block_m, int block_n, int dtype,
                     int* path, int* tile_m, int* tile_n);

/*
 * Number of work items rsfa_fwd splits this problem into: (batch, head, block of query rows) units
 * that the persistent tcgen05 kernels hand out through their queue (256 rows each, 128 at D = 256; the
 * forms for small launches, see rsfa_fwd, deal out the same rows in other portions),
 * or the CTAs of the short-sequence kernel (64 rows each, all on grid.x, so the count may exceed
 * 65535).  Counterpart of NUM_BLOCKS = cdiv(N_CTX, BLOCK_M) * Z * H (:289-294).  Needs no device.
 */
RSFA_API int rsfa_work_items(int B, int H, int S, int D, int causal, float sm_scale, long long* items);

/*
 * Number of streaming multiprocessors of a device: the grid size of the persistent kernel.
 * Replaces get_num_compute_cores (:19-21).  Returns the count (> 0) or a negative error.
 */
RSFA_API int rsfa_sm_count(int device);

/*
 * Synchronise `device` and return the status word its kernels share (this call allocates nothing
 * and reads only the scratch that rsfa_fwd or rsfa_fwd_noalloc has already set up on the device): RSFA_OK, or
 * RSFA_ERR_DEVICE_STATUS with the raw word in *raw (if not NULL): (1 << 16) | tag, where tag names
 * the wait that ran out (40: a load of rsfa_cache4_attention), or (2 << 16) | tag, see above, for an
 * index out of range.  Reading clears the word.  rsfa_fwd itself returns RSFA_OK for a call whose kernel later gives up (the launch is asynchronous) and the output of that call is then
 * incomplete: callers that care call this function at their synchronisation points, or set the
 * "check_status" option, under which every rsfa_fwd copies the word to the host behind its kernels
 * and the next rsfa_fwd on that device returns RSFA_ERR_DEVICE_STATUS without launching once a
 * non-zero word has arrived (this function then reports and clears it).
 * The reference has no counterpart: its kernels cannot time out.
 */
RSFA_API int rsfa_device_status(int device, int* raw);

/* Count of kernels this library has launched in this process (all devices). */
RSFA_API long long rsfa_launch_count(void);

/*
 * Tuning / test knobs.  Names: "force_path" (-1 auto, 0 generic, 1 tcgen05),
 * "wait_limit_ms" (bound of every in-kernel wait, default 2000), "tcgen05_variant" (-1: by size,
 * see block_m / block_n of rsfa_fwd; 0 / 1 force the pair form of the single-buffered 128-key /
 * double-buffered 64-key kernel for D <= 128; 2 forces 128-key tiles with the separate-P kernel where
 * it exists), "host_slab_heads"
 * (heads per staging slab of rsfa_fwd_host, 0 = automatic), "pdl" (1, the default: the tcgen05 kernels
 * are launched with programmatic stream serialisation, so the set-up of a launch overlaps the tail of
 * the kernel in front of it on the stream; they wait for that kernel before touching global memory),
 * "check_status" (0 / 1, see rsfa_device_status), "test_drop_load" (-1 = off; n >= 0: every CTA of the
 * 128-key tcgen05 kernel leaves out its n-th K/V tile load and the barrier arrival that announces it, and
 * the kernel for a single key tile, of the loads that it starts with, those of the heads from n on (of B * H),
 * and every warp of rsfa_cache4_attention its n-th tile of the cache, so that a bounded wait runs out - for
 * tests of the wait-expired path; the output of such a call is incomplete).
 * rsfa_get_option also answers "workspace_devices": the number of devices on which rsfa_fwd has
 * created its workspace (0 in a process that has only used rsfa_fwd_noalloc).
 * Unknown names -> RSFA_ERR_INVALID_ARGUMENT.
 */
RSFA_API int rsfa_set_option(const char* name, long long value);
RSFA_API long long rsfa_get_option(const char* name);

RSFA_API const char* rsfa_strerror(int code);

/* major*10000 + minor*100 + patch */
RSFA_API int rsfa_version(void);

#ifdef __cplusplus
}
#endif
#endif /* RSFA_H_ */
