// What the paged-cache kernels share: argument checks, element types, where a row or a page is.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>

namespace {

// ---- element types ----
__host__ __device__ constexpr int type_size(int t) { return t == B200Q_F32 ? 4 : 2; }
static inline bool type_known(int t) { return t == B200Q_F32 || t == B200Q_F16 || t == B200Q_BF16; }

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ uint32_t pack2(float a, float b, int type) {      // two 16-bit values, rounded to nearest
  if (type == B200Q_F16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float load_as_f(const void* base, int type, int64_t i) {
  return type == B200Q_F32 ? static_cast<const float*>(base)[i] : type == B200Q_F16 ? __half2float(static_cast<const __half*>(base)[i])
                                                                                   : __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
}
__device__ __forceinline__ void store_as(void* base, int type, int64_t i, float v) {
  if (type == B200Q_F32) static_cast<float*>(base)[i] = v;
  else if (type == B200Q_F16) static_cast<__half*>(base)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
}

// Division of values below 2^31 by a number that the host knows: n / d = (high word of n * mul + n) >> shift (a division proper is forty dependent instructions)
struct Divisor {
  uint32_t mul, shift;
  __device__ __forceinline__ int div(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
};
static inline Divisor divisor_of(int d) {
  uint32_t shift = 0;
  while ((1u << shift) < (uint32_t)d) shift++;      // d <= 2^shift < 2 d; mul = 2^32 (2^shift - d) / d + 1
  return Divisor{(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1), shift};
}

// ---- tables ----
struct PagedTables {
  const int32_t *row_off, *length, *pages;
  int n_seqs, table_stride, n_rows, max_new, max_len, n_pages, page_size;
};

// The sequence of a row, its rows and its length, by a whole warp; begin > row: of no sequence.  One token of every sequence is the usual case of large batches and asked first; up to 32 sequences are
// asked all at once, so that this is one load's latency either way.
struct SeqOfRow { int seq, begin, end, length; };
__device__ __forceinline__ SeqOfRow seq_of_row(const PagedTables& t, int row) {
  const int lane = threadIdx.x & 31;
  if (t.n_seqs > 32) {
    const int g = min(row, t.n_seqs - 1);
    const SeqOfRow w{g, t.row_off[g], t.row_off[g + 1], t.length[g]};
    if (w.begin <= row && row < w.end) return w;
  }
  for (int s0 = 0; s0 < t.n_seqs; s0 += 32) {
    int b = 0, e = 0, l = 0;
    if (s0 + lane < t.n_seqs) { b = t.row_off[s0 + lane]; e = t.row_off[s0 + lane + 1]; l = t.length[s0 + lane]; }
    const unsigned here = __ballot_sync(0xffffffffu, b <= row && row < e);
    if (here) {
      const int src = __ffs(here) - 1;
      return SeqOfRow{s0 + src, __shfl_sync(0xffffffffu, b, src), __shfl_sync(0xffffffffu, e, src), __shfl_sync(0xffffffffu, l, src)};
    }
  }
  return SeqOfRow{0, INT32_MAX, 0, 0};
}

// ---- checks of what all entry points take ----
static inline int check_cache(const b200q_paged_cache* c) {
  if (!c || !c->k || !c->v || !type_known(c->dtype) || c->n_pages <= 0 || c->page_size <= 0 || c->n_kv_heads <= 0) return B200Q_ERR_BAD_ARG;
  if (c->head_dim != 16 && c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return B200Q_ERR_BAD_SHAPE;
  const int64_t unit = 16 / type_size(c->dtype);
  if (c->page_stride < c->head_dim || c->head_stride < c->head_dim || c->row_stride < c->head_dim) return B200Q_ERR_BAD_SHAPE;
  if (c->page_stride % unit || c->head_stride % unit || c->row_stride % unit || (((uintptr_t)c->k | (uintptr_t)c->v) & 15)) return B200Q_ERR_MISALIGNED;
  return B200Q_OK;
}
static inline int check_batch(const b200q_paged_batch* b) {
  if (!b || b->n_seqs < 0 || b->n_rows < 0 || b->max_new < 0 || b->max_len < 0) return B200Q_ERR_BAD_ARG;
  if (b->n_seqs == 0 || b->n_rows == 0) return B200Q_OK;
  if (!b->row_off || !b->length || !b->pages || b->table_stride <= 0 || b->max_new <= 0) return B200Q_ERR_BAD_ARG;
  if (((uintptr_t)b->row_off | (uintptr_t)b->length | (uintptr_t)b->pages) & 3) return B200Q_ERR_MISALIGNED;
  return B200Q_OK;
}
static inline PagedTables tables_of(const b200q_paged_cache* c, const b200q_paged_batch* b) {
  return PagedTables{b->row_off, b->length, b->pages, b->n_seqs, b->table_stride, b->n_rows, b->max_new, b->max_len, c->n_pages, c->page_size};
}

}  // namespace
