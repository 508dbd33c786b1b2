// C entry points of the operators around attention: rotary positions and the paged 4-bit cache.  Arguments are
// checked here, on the host; what lies in device memory (positions, pages, lengths) is checked by the kernels.
// include/rsfa.h has the contract of every function.
#include <cmath>
#include <cstring>

#include "../../include/rsfa.h"
#include "common.cuh"

namespace {

constexpr long long kMostInt = 2147483647LL;
constexpr double kMostTiles = 1099511627776.0;   // 2^40, over a thousand warps of a B200 and more

bool valid_dtype(int dtype) { return dtype == RSFA_DTYPE_F16 || dtype == RSFA_DTYPE_BF16; }
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// A dense [B, H, S, D] tensor whose rows are read 16 bytes at a time.
bool valid_tensor(const void* p, const int64_t* st, int B, int H, int S, int D) {
  if (p == nullptr || !aligned(p, 16) || st[3] != 1) return false;
  const int extent[3] = {B, H, S};
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && (st[i] < D || (st[i] & 7) != 0)) return false;
  return true;
}

// The cache's own arguments, in the form the kernels take.
int take_cache(const rsfa_cache4* in, rsfa::Cache4* c) {
  if (in == nullptr || in->kv == nullptr || in->table == nullptr || in->lengths == nullptr) return RSFA_ERR_INVALID_ARGUMENT;
  if (in->batch < 1 || in->heads < 1 || in->pages < 1 || in->max_pages < 1 || !valid_dtype(in->dtype)) return RSFA_ERR_INVALID_ARGUMENT;
  if (in->head_dim == 16 || in->head_dim == 32) return RSFA_ERR_UNSUPPORTED;
  if (in->head_dim != 64 && in->head_dim != 128 && in->head_dim != 256) return RSFA_ERR_INVALID_ARGUMENT;
  int shift = 4;
  while (shift < 10 && (1 << shift) != in->page_size) ++shift;
  if ((1 << shift) != in->page_size) return RSFA_ERR_INVALID_ARGUMENT;      // 16 ... 1024
  if (static_cast<long long>(in->max_pages) << shift > 1LL << 30) return RSFA_ERR_TOO_LARGE;
  const int64_t rows = static_cast<int64_t>(in->page_size);
  const int64_t bytes = rows * (in->head_dim * 5 / 4);
  if (!aligned(in->kv, 16) || (in->kv_stride[0] & 15) != 0 || (in->kv_stride[1] & 15) != 0) return RSFA_ERR_INVALID_ARGUMENT;
  if ((in->pages > 1 && in->kv_stride[0] < bytes) || (in->heads > 1 && in->kv_stride[1] < bytes)) return RSFA_ERR_INVALID_ARGUMENT;
  if (!aligned(in->table, 4) || !aligned(in->lengths, 4) || !aligned(in->weight, 4) || !aligned(in->position, 4)) return RSFA_ERR_INVALID_ARGUMENT;
  if (in->batch > 1 && in->table_stride < 0) return RSFA_ERR_INVALID_ARGUMENT;
  const void* extra[2] = {in->weight, in->position};
  const int64_t* extra_stride[2] = {in->weight_stride, in->position_stride};
  for (int i = 0; i < 2; ++i)
    if (extra[i] != nullptr && ((in->pages > 1 && extra_stride[i][0] < rows) || (in->heads > 1 && extra_stride[i][1] < rows)))
      return RSFA_ERR_INVALID_ARGUMENT;
  c->kv = static_cast<uint8_t*>(in->kv);
  c->weight = in->weight;
  c->position = in->position;
  c->table = in->table;
  c->lengths = in->lengths;
  for (int i = 0; i < 2; ++i) {
    c->kv_stride[i] = in->kv_stride[i];
    c->weight_stride[i] = in->weight_stride[i];
    c->position_stride[i] = in->position_stride[i];
  }
  c->table_stride = in->table_stride;
  c->B = in->batch;
  c->H = in->heads;
  c->D = in->head_dim;
  c->pages = in->pages;
  c->max_pages = in->max_pages;
  c->page_shift = shift;
  c->bf16 = in->dtype == RSFA_DTYPE_BF16 ? 1 : 0;
  return RSFA_OK;
}

int take_rows(const rsfa::Cache4& c, void* k, void* v, int S, const int64_t* strides, rsfa::Cache4Rows* r) {
  if (S < 1 || strides == nullptr || !valid_tensor(k, strides, c.B, c.H, S, c.D) || !valid_tensor(v, strides + 4, c.B, c.H, S, c.D))
    return RSFA_ERR_INVALID_ARGUMENT;
  if (static_cast<double>(c.B) * c.H * S > static_cast<double>(kMostInt)) return RSFA_ERR_TOO_LARGE;
  std::memset(r, 0, sizeof(*r));
  r->k = k;
  r->v = v;
  r->S = S;
  for (int i = 0; i < 3; ++i) {
    r->k_stride[i] = strides[i];
    r->v_stride[i] = strides[4 + i];
  }
  return RSFA_OK;
}

// Query rows of all heads are counted in 32 bits, and so is a warp's share of all tiles (of 32 tokens or more, for 8 query rows
// or more).
bool countable(const rsfa::Cache4& c, int q_heads, int S) {
  const double tiles = std::ceil(static_cast<double>(c.max_pages) * (1 << c.page_shift) / 32.0) + 2.0;
  return static_cast<double>(c.B) * q_heads * S <= static_cast<double>(kMostInt) &&
         c.B * std::ceil(static_cast<double>(q_heads / c.H) * S / 8.0) * c.H * tiles <= kMostTiles;
}

// Heads of all sequences are counted in 32 bits, the bytes of their moves in 64.
bool movable(int batch, int heads, int most_moves) {
  const double all = static_cast<double>(batch) * heads;
  return all <= static_cast<double>(kMostInt) && all * (2.0 * most_moves + 2.0) * sizeof(int) < 9.0e18;
}

}  // namespace

extern "C" {

int rsfa_rotary_table(float* table, int length, int dim, double base, int scaling, double factor, int original_length,
                      double low_turns, double high_turns, double multiplier, void* stream) {
  if (table == nullptr || !aligned(table, 16) || length < 1 || dim < 2 || dim > 256 || (dim & 1) != 0) return RSFA_ERR_INVALID_ARGUMENT;
  if (!(base > 1.0) || !std::isfinite(base) || !std::isfinite(multiplier)) return RSFA_ERR_INVALID_ARGUMENT;
  if (scaling < RSFA_ROTARY_NONE || scaling > RSFA_ROTARY_BANDS) return RSFA_ERR_INVALID_ARGUMENT;
  if (scaling != RSFA_ROTARY_NONE && (!(factor > 0.0) || !std::isfinite(factor))) return RSFA_ERR_INVALID_ARGUMENT;
  if ((scaling == RSFA_ROTARY_YARN || scaling == RSFA_ROTARY_BANDS) &&
      (original_length < 1 || !(low_turns > 0.0) || !(high_turns > low_turns) || !std::isfinite(high_turns)))
    return RSFA_ERR_INVALID_ARGUMENT;
  rsfa::CallScratch d;
  const int rc = rsfa::begin_call(&d);
  if (rc != RSFA_OK) return rc;
  const double args[6] = {base, factor, static_cast<double>(original_length), low_turns, high_turns, multiplier};
  long long launches = 0;
  const cudaError_t e = rsfa::launch_rotary_table(table, length, dim, args, scaling, static_cast<cudaStream_t>(stream), &launches);
  return rsfa::end_call(d, static_cast<cudaStream_t>(stream), e, launches);
}

int rsfa_rotary(const void* q, const void* k, void* q_out, void* k_out, int B, int Hq, int Hk, int S, int D,
                const int64_t* strides, const float* table, int table_length, int rotary_dim, const void* positions,
                int positions_64, const int64_t* position_strides, int interleaved, int inverse, int dtype, void* stream) {
  if (strides == nullptr || table == nullptr || !valid_dtype(dtype)) return RSFA_ERR_INVALID_ARGUMENT;
  if (B < 1 || Hq < 1 || Hk < 0 || S < 1 || (Hk > 0) != (k != nullptr)) return RSFA_ERR_INVALID_ARGUMENT;
  if (D != 16 && D != 32 && D != 64 && D != 128 && D != 256) return RSFA_ERR_INVALID_ARGUMENT;
  if (rotary_dim < 2 || rotary_dim > D || (rotary_dim & 1) != 0 || table_length < 1 || !aligned(table, 8)) return RSFA_ERR_INVALID_ARGUMENT;
  if (!valid_tensor(q, strides, B, Hq, S, D) || !valid_tensor(q_out, strides + 8, B, Hq, S, D)) return RSFA_ERR_INVALID_ARGUMENT;
  if (Hk > 0 && (!valid_tensor(k, strides + 4, B, Hk, S, D) || !valid_tensor(k_out, strides + 12, B, Hk, S, D))) return RSFA_ERR_INVALID_ARGUMENT;
  if (positions != nullptr && (position_strides == nullptr || !aligned(positions, positions_64 ? 8 : 4))) return RSFA_ERR_INVALID_ARGUMENT;
  // a thread of every chunk of a position is numbered in 32 bits, heads are on the grid's second axis
  if (static_cast<double>(B) * S * (D / 2) > static_cast<double>(kMostInt) || static_cast<long long>(Hq) + Hk > 65535) return RSFA_ERR_TOO_LARGE;
  rsfa::CallScratch d;
  const int rc = rsfa::begin_call(&d);
  if (rc != RSFA_OK) return rc;
  rsfa::RotaryParams p;
  std::memset(&p, 0, sizeof(p));
  p.x[0] = q;
  p.x[1] = k;
  p.y[0] = q_out;
  p.y[1] = k_out;
  for (int t = 0; t < (Hk > 0 ? 2 : 1); ++t)
    for (int i = 0; i < 3; ++i) {
      p.x_stride[t][i] = strides[4 * t + i];
      p.y_stride[t][i] = strides[8 + 4 * t + i];
    }
  p.heads[0] = Hq;
  p.heads[1] = Hk;
  p.table = table;
  p.positions = positions;
  p.positions_64 = positions_64;
  if (positions != nullptr) {
    p.pos_stride[0] = position_strides[0];
    p.pos_stride[1] = position_strides[1];
  }
  p.B = B;
  p.S = S;
  p.D = D;
  p.R = rotary_dim;
  p.table_length = table_length;
  p.interleaved = interleaved;
  p.inverse = inverse;
  p.bf16 = dtype == RSFA_DTYPE_BF16 ? 1 : 0;
  p.status = d.status;
  long long launches = 0;
  const cudaError_t e = rsfa::launch_rotary(p, d.sm_count, static_cast<cudaStream_t>(stream), &launches);
  return rsfa::end_call(d, static_cast<cudaStream_t>(stream), e, launches);
}

int rsfa_cache4_append(const rsfa_cache4* cache, const void* k, const void* v, int S, const int64_t* strides, const int* counts,
                       const int* positions, const int64_t* position_strides, void* stream) {
  rsfa::Cache4 c;
  int rc = take_cache(cache, &c);
  if (rc != RSFA_OK) return rc;
  rsfa::Cache4Rows r;
  rc = take_rows(c, const_cast<void*>(k), const_cast<void*>(v), S, strides, &r);
  if (rc != RSFA_OK) return rc;
  if (!aligned(counts, 4) || !aligned(positions, 4) || (positions != nullptr && position_strides == nullptr)) return RSFA_ERR_INVALID_ARGUMENT;
  if ((positions != nullptr) != (c.position != nullptr)) return RSFA_ERR_INVALID_ARGUMENT;
  r.counts = counts;
  r.positions = positions;
  if (positions != nullptr) {
    r.positions_stride[0] = position_strides[0];
    r.positions_stride[1] = position_strides[1];
  }
  rsfa::CallScratch d;
  rc = rsfa::begin_call(&d);
  if (rc != RSFA_OK) return rc;
  c.status = d.status;
  long long launches = 0;
  const cudaError_t e = rsfa::launch_cache4_append(c, r, static_cast<cudaStream_t>(stream), &launches);
  return rsfa::end_call(d, static_cast<cudaStream_t>(stream), e, launches);
}

int rsfa_cache4_read(const rsfa_cache4* cache, void* k, void* v, int N, const int64_t* strides, const int* starts, void* stream) {
  rsfa::Cache4 c;
  int rc = take_cache(cache, &c);
  if (rc != RSFA_OK) return rc;
  rsfa::Cache4Rows r;
  rc = take_rows(c, k, v, N, strides, &r);
  if (rc != RSFA_OK) return rc;
  if (!aligned(starts, 4)) return RSFA_ERR_INVALID_ARGUMENT;
  r.starts = starts;
  rsfa::CallScratch d;
  rc = rsfa::begin_call(&d);
  if (rc != RSFA_OK) return rc;
  c.status = d.status;
  long long launches = 0;
  const cudaError_t e = rsfa::launch_cache4_read(c, r, static_cast<cudaStream_t>(stream), &launches);
  return rsfa::end_call(d, static_cast<cudaStream_t>(stream), e, launches);
}

long long rsfa_cache4_attention_workspace(const rsfa_cache4* cache, int q_heads, int S) {
  rsfa::Cache4 c;
  const int rc = take_cache(cache, &c);
  if (rc != RSFA_OK) return rc;
  if (q_heads < c.H || q_heads % c.H != 0 || S < 1) return RSFA_ERR_INVALID_ARGUMENT;
  if (!countable(c, q_heads, S)) return RSFA_ERR_TOO_LARGE;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) {
    cudaGetLastError();
    return RSFA_ERR_NO_DEVICE;
  }
  const int sms = rsfa_sm_count(device);
  if (sms <= 0) return sms;
  return static_cast<long long>(rsfa::cache4_attention_workspace(c, q_heads, S, sms).total);
}

int rsfa_cache4_attention(const rsfa_cache4* cache, const void* q, void* o, float* lse, int q_heads, int S, const int64_t* strides,
                          const int* counts, float sm_scale, void* workspace, long long workspace_bytes, void* stream) {
  rsfa::Cache4 c;
  int rc = take_cache(cache, &c);
  if (rc != RSFA_OK) return rc;
  if (q_heads < c.H || q_heads % c.H != 0 || S < 1 || strides == nullptr || !(sm_scale == sm_scale)) return RSFA_ERR_INVALID_ARGUMENT;
  if (!valid_tensor(q, strides, c.B, q_heads, S, c.D) || !valid_tensor(o, strides + 4, c.B, q_heads, S, c.D)) return RSFA_ERR_INVALID_ARGUMENT;
  if (!aligned(lse, 4) || !aligned(counts, 4) || (c.weight != nullptr && lse == nullptr)) return RSFA_ERR_INVALID_ARGUMENT;
  if (!countable(c, q_heads, S)) return RSFA_ERR_TOO_LARGE;
  rsfa::CallScratch d;
  rc = rsfa::begin_call(&d);
  if (rc != RSFA_OK) return rc;
  const rsfa::Cache4Workspace need = rsfa::cache4_attention_workspace(c, q_heads, S, d.sm_count);
  if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < static_cast<long long>(need.total)) return RSFA_ERR_INVALID_ARGUMENT;
  c.status = d.status;
  rsfa::Cache4Attention a;
  std::memset(&a, 0, sizeof(a));
  a.q = q;
  a.o = o;
  a.lse = lse;
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = strides[i];
    a.o_stride[i] = strides[4 + i];
  }
  a.Hq = q_heads;
  a.S = S;
  a.counts = counts;
  a.sm_scale = sm_scale;
  a.pieces = static_cast<float*>(workspace);
  a.scores = a.pieces + need.pieces / sizeof(float);
  long long launches = 0;
  const cudaError_t e = rsfa::launch_cache4_attention(c, a, d.sm_count, static_cast<cudaStream_t>(stream), &launches);
  return rsfa::end_call(d, static_cast<cudaStream_t>(stream), e, launches);
}

long long rsfa_cache4_evict_workspace(int batch, int heads, int most_moves) {
  if (batch < 1 || heads < 1 || most_moves < 0) return RSFA_ERR_INVALID_ARGUMENT;
  if (!movable(batch, heads, most_moves)) return RSFA_ERR_TOO_LARGE;
  return static_cast<long long>(rsfa::cache4_evict_workspace(batch, heads, most_moves));
}

int rsfa_cache4_evict(const rsfa_cache4* cache, int budget, int recent, int* new_lengths, void* workspace, long long workspace_bytes,
                      void* stream) {
  rsfa::Cache4 c;
  int rc = take_cache(cache, &c);
  if (rc != RSFA_OK) return rc;
  if (c.weight == nullptr || c.position == nullptr || new_lengths == nullptr || new_lengths == c.lengths) return RSFA_ERR_INVALID_ARGUMENT;
  if (budget < 1 || recent < 0 || recent > budget || !aligned(new_lengths, 4)) return RSFA_ERR_INVALID_ARGUMENT;
  const int most_moves = rsfa::cache4_most_moves(c, budget);
  if (!movable(c.B, c.H, most_moves)) return RSFA_ERR_TOO_LARGE;
  if (workspace == nullptr || !aligned(workspace, 16) ||
      workspace_bytes < static_cast<long long>(rsfa::cache4_evict_workspace(c.B, c.H, most_moves)))
    return RSFA_ERR_INVALID_ARGUMENT;
  rsfa::CallScratch d;
  rc = rsfa::begin_call(&d);
  if (rc != RSFA_OK) return rc;
  c.status = d.status;
  rsfa::Cache4Evict e;
  e.budget = budget;
  e.recent = recent;
  e.most_moves = most_moves;
  e.new_lengths = new_lengths;
  e.moves = static_cast<int*>(workspace);
  long long launches = 0;
  const cudaError_t err = rsfa::launch_cache4_evict(c, e, d.sm_count, static_cast<cudaStream_t>(stream), &launches);
  return rsfa::end_call(d, static_cast<cudaStream_t>(stream), err, launches);
}

}  // extern "C"
