// New tokens on their way into a paged KV cache: the norms of the query and key heads, the position rotation and the store, in one pass over the projections.
//   head x of dim values, x' = x / sqrt(mean(x^2) + eps) * w (where a norm is asked for); rotated: (a, b) = (x'[d], x'[d + r/2]) -> (a cos - b sin, b cos + a sin), d < r/2
//   (tinygrad/nn/__init__.py:300-304, tinygrad/llm/model.py:29-33); q heads go to rows again, k and v heads to slot p % page_size of the page of position p (model.py:200-207).
// Bound by memory: every value is read once and written once.  A thread owns both members of its pairs, 16 bytes each, so the rotation needs no exchange and the norm
// a shuffle sum over the threads of a head (16 for 128 fp32 values); a CTA has one row, whose cosines, sines and place are looked up while the values are on their way.
#include "paged.cuh"
#include <algorithm>

namespace {

__device__ int g_paged_status = 0;      // 2: a position or page of the tables does not exist

struct RowsParams {
  const void* x;
  void* q;                       // rows of query heads (append), or of query and key heads (norms alone)
  void *k, *v;                   // pages; NULL: norms alone
  int q_dtype, kv_dtype;
  int64_t x_stride, q_stride, page_stride, head_stride, row_stride;
  int n_heads, n_kv, heads;      // heads: those of a row that are read
  float eps;
  const __half *q_norm, *k_norm;
  const float* rope;
  int rope_dim, rope_len;
  const int32_t* positions;      // norms alone
  Divisor by_page;
  PagedTables t;
};

constexpr int ROW_THREADS = 256, MANY_THREADS = 148 * 2048;

// VEC values of type X from p
template <typename X, int VEC> struct Raw { uint4 v; };
template <typename X> struct Raw<X, 1> { X v; };
template <typename X, int VEC> __device__ __forceinline__ void unpack(const Raw<X, VEC>& r, float (&f)[VEC]) {
  if constexpr (VEC == 1) f[0] = to_f(r.v);
  else {
    const X* e = reinterpret_cast<const X*>(&r.v);
#pragma unroll
    for (int i = 0; i < VEC; i++) f[i] = to_f(e[i]);
  }
}
template <typename X, int VEC> __device__ __forceinline__ Raw<X, VEC> load_raw(const X* p) {
  Raw<X, VEC> r;
  if constexpr (VEC == 1) r.v = *p;
  else r.v = *reinterpret_cast<const uint4*>(p);
  return r;
}
template <int VEC> __device__ __forceinline__ void store_vec(void* base, int type, int64_t i, const float (&f)[VEC]) {
  if constexpr (VEC == 1) store_as(base, type, i, f[0]);
  else if (type == B200Q_F32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
#pragma unroll
    for (int j = 0; j < VEC / 4; j++) d[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
  } else {
    uint32_t w[VEC / 2];
    if (type == B200Q_F16) {
#pragma unroll
      for (int j = 0; j < VEC / 2; j++) w[j] = pack2(f[2 * j], f[2 * j + 1], B200Q_F16);
    } else {
#pragma unroll
      for (int j = 0; j < VEC / 2; j++) w[j] = pack2(f[2 * j], f[2 * j + 1], B200Q_BF16);
    }
    void* d = static_cast<uint16_t*>(base) + i;
    if constexpr (VEC == 8) *static_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
    else *static_cast<uint2*>(d) = make_uint2(w[0], w[1]);
  }
}

// VEC values of a table on 16-byte (fp32) or 2 VEC-byte (fp16) boundaries
template <int VEC> __device__ __forceinline__ void load_table(const float* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) f[0] = *p;
  else
#pragma unroll
    for (int j = 0; j < VEC; j += 4) { const float4 v = *reinterpret_cast<const float4*>(p + j); f[j] = v.x; f[j + 1] = v.y; f[j + 2] = v.z; f[j + 3] = v.w; }
}
template <int VEC> __device__ __forceinline__ void load_table(const __half* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) f[0] = __half2float(*p);
  else {
    uint32_t w[VEC / 2];
    if constexpr (VEC == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int j = 0; j < VEC / 2; j++) { const float2 v = __half22float2(*reinterpret_cast<const __half2*>(w + j)); f[2 * j] = v.x; f[2 * j + 1] = v.y; }
  }
}

// Where a row's position is: its entry in the pages (-1: none), whether its heads are zeros, whether it belongs to a sequence.  By a whole warp.
struct RowPlace { int64_t at; int pos; bool zero, none; };
__device__ __forceinline__ RowPlace place_of_row(const RowsParams& p, int row) {
  RowPlace w{-1, 0, false, false};
  bool bad = false;
  if (p.k) {
    const SeqOfRow s = seq_of_row(p.t, row);
    if (s.begin > row) { w.none = true; return w; }
    w.pos = s.length - (s.end - row);
    const int index = w.pos < 0 ? 0 : p.by_page.div(w.pos);
    if (w.pos >= 0 && index < p.t.table_stride) {
      const int page = p.t.pages[(int64_t)s.seq * p.t.table_stride + index];
      if (page >= 0 && page < p.t.n_pages) w.at = page * p.page_stride + (w.pos - index * p.t.page_size) * p.row_stride;
    }
    bad = w.at < 0;
  } else if (p.rope) w.pos = p.positions[row];
  w.zero = p.rope && (w.pos < 0 || w.pos >= p.rope_len);
  if ((bad || w.zero) && (threadIdx.x & 31) == 0) atomicExch(&g_paged_status, 2);
  if (w.zero) w.at = -1;
  return w;
}

// A head's pairs: TPH threads, NG groups of VEC pairs each.
template <int D, int VEC> struct Pairs {
  static constexpr int ALL = D / 2 / VEC, TPH = ALL < 32 ? ALL : 32, NG = ALL / TPH;
  int da[NG], db[NG];                // where the group's first members and their partners are
  int half;
  __device__ __forceinline__ Pairs(const RowsParams& p, int sub) {
    half = p.rope ? p.rope_dim / 2 : 0;
    const int rest = (D - 2 * half) / 2;
#pragma unroll
    for (int g = 0; g < NG; g++) {
      const int i = (g * TPH + sub) * VEC;
      da[g] = i < half ? i : half + i;
      db[g] = da[g] + (i < half ? half : rest);
    }
  }
};
// cosines and sines of a thread's pairs
template <int D, int VEC>
__device__ __forceinline__ void load_angles(const RowsParams& p, const Pairs<D, VEC>& w, const RowPlace& at, float (&c)[Pairs<D, VEC>::NG][VEC], float (&s)[Pairs<D, VEC>::NG][VEC]) {
#pragma unroll
  for (int g = 0; g < Pairs<D, VEC>::NG; g++)
    if (!at.zero && w.da[g] < w.half) {
      load_table<VEC>(p.rope + (int64_t)at.pos * p.rope_dim + w.da[g], c[g]);
      load_table<VEC>(p.rope + (int64_t)at.pos * p.rope_dim + w.db[g], s[g]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++) { c[g][j] = 1.f; s[g][j] = 0.f; }
    }
}
// One head h of a row, its pairs in a and b: norm, rotation, store.  Whole warps take part (h may be past the last head).
template <int D, int VEC>
__device__ __forceinline__ void do_head(const RowsParams& p, const Pairs<D, VEC>& w, const RowPlace& at, int row, int h, float (&a)[Pairs<D, VEC>::NG][VEC], float (&b)[Pairs<D, VEC>::NG][VEC],
                                        const float (&c)[Pairs<D, VEC>::NG][VEC], const float (&s)[Pairs<D, VEC>::NG][VEC]) {
  constexpr int NG = Pairs<D, VEC>::NG;
  const bool is_q = h < p.n_heads, is_k = !is_q && h < p.n_heads + p.n_kv;
  if (p.q_norm || p.k_norm) {
    float ss = 0.f;
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
      for (int j = 0; j < VEC; j++) ss = fmaf(a[g][j], a[g][j], fmaf(b[g][j], b[g][j], ss));
#pragma unroll
    for (int o = Pairs<D, VEC>::TPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const __half* wn = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
    if (wn) {
      const float r = rsqrtf(ss * (1.f / D) + p.eps);      // (within two units of the last place; with a root and a quotient 4096 rows took 1 us more: instructions are half of what bounds this)
#pragma unroll
      for (int g = 0; g < NG; g++) {
        float wa[VEC], wb[VEC];
        load_table<VEC>(wn + w.da[g], wa);
        load_table<VEC>(wn + w.db[g], wb);
#pragma unroll
        for (int j = 0; j < VEC; j++) { a[g][j] *= r * wa[j]; b[g][j] *= r * wb[j]; }
      }
    }
  }
  if (h >= p.heads) return;
#pragma unroll
  for (int g = 0; g < NG; g++) {
    if (is_q || is_k) {
      if (w.da[g] < w.half) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const float u = a[g][j], v = b[g][j];
          a[g][j] = u * c[g][j] - v * s[g][j];
          b[g][j] = v * c[g][j] + u * s[g][j];
        }
      }
      if (at.zero) {
#pragma unroll
        for (int j = 0; j < VEC; j++) a[g][j] = b[g][j] = 0.f;
      }
    }
    if (is_q || !p.k) {
      const int64_t o = row * p.q_stride + h * D;
      store_vec<VEC>(p.q, p.q_dtype, o + w.da[g], a[g]);
      store_vec<VEC>(p.q, p.q_dtype, o + w.db[g], b[g]);
    } else if (at.at >= 0) {
      void* pool = is_k ? p.k : p.v;
      const int64_t o = at.at + (h - p.n_heads - (is_k ? 0 : p.n_kv)) * p.head_stride;
      store_vec<VEC>(pool, p.kv_dtype, o + w.da[g], a[g]);
      store_vec<VEC>(pool, p.kv_dtype, o + w.db[g], b[g]);
    }
  }
}

// A CTA has ROWS rows; a thread IT heads of each, blockDim / TPH apart.  All of its loads are asked for before the rows' places are looked up.
template <typename X, int D, int VEC, int IT, int ROWS>
__global__ void __launch_bounds__(ROW_THREADS, IT == 1 && ROWS == 1 ? 6 : IT <= 3 && ROWS == 1 ? 5 : 4) rows_to_heads_kernel(const RowsParams p, int n_rows) {
  constexpr int TPH = Pairs<D, VEC>::TPH, NG = Pairs<D, VEC>::NG;
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = blockIdx.x * ROWS, slots = blockDim.x / TPH, h0 = blockIdx.y * (slots * IT) + threadIdx.x / TPH;
  const Pairs<D, VEC> w(p, threadIdx.x % TPH);
  Raw<X, VEC> ra[ROWS][IT][NG], rb[ROWS][IT][NG];
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const X* x = static_cast<const X*>(p.x) + min(row0 + i, n_rows - 1) * p.x_stride;
#pragma unroll
    for (int t = 0; t < IT; t++)
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const X* y = x + min(h0 + t * slots, p.heads - 1) * D;
        ra[i][t][g] = load_raw<X, VEC>(y + w.da[g]);
        rb[i][t][g] = load_raw<X, VEC>(y + w.db[g]);
      }
  }
  RowPlace at[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    if (row0 + i < n_rows) at[i] = place_of_row(p, row0 + i);
    else at[i].none = true;
  }
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    if (at[i].none) continue;
    float c[NG][VEC], s[NG][VEC];
    load_angles<D, VEC>(p, w, at[i], c, s);
#pragma unroll
    for (int t = 0; t < IT; t++) {
      float a[NG][VEC], b[NG][VEC];
#pragma unroll
      for (int g = 0; g < NG; g++) { unpack<X, VEC>(ra[i][t][g], a[g]); unpack<X, VEC>(rb[i][t][g], b[g]); }
      do_head<D, VEC>(p, w, at[i], row0 + i, h0 + t * slots, a, b, c, s);
    }
  }
}

// Few rows: a head a thread group.  Many: all heads of a row (of two rows, where nothing has to be looked up) in a CTA, with up to four heads a thread.  us, 4096 rows of 48 fp32 heads of 128,
// normed, / 4017 of 48 bf16 heads of 64 / norms alone of 8191 x 32 fp16 heads of 128: three heads a thread and five CTAs an SM 37.5 / - / -, one head and six / four 43.7, - / 14.8, 16.6 / 30.9, 29.9, two rows
// and four CTAs - / 16.6 / 27.8, four rows and two CTAs - / 25.0 / 39.3; rows streamed through shared memory by bulk copies, a warp looking up places ahead, 42.6 / 21.2 / 35.2.
template <typename X, int D, int VEC>
int launch_vec(const RowsParams& p, int n_rows, bool pdl, cudaStream_t st) {
  constexpr int TPH = Pairs<D, VEC>::TPH;
  const int threads = p.heads * TPH, it = (int64_t)n_rows * threads > MANY_THREADS ? std::min(4, ceil_div(threads, ROW_THREADS)) : 0;
  const int block = it == 0 ? ROW_THREADS : std::min(ROW_THREADS, ceil_div(ceil_div(p.heads, it) * TPH, 32) * 32), rows = it == 1 && !p.k ? 2 : 1;
  auto kernel = it == 2 ? rows_to_heads_kernel<X, D, VEC, 2, 1> : it == 3 ? rows_to_heads_kernel<X, D, VEC, 3, 1> : it == 4 ? rows_to_heads_kernel<X, D, VEC, 4, 1>
                : rows == 2 ? rows_to_heads_kernel<X, D, VEC, 1, 2> : rows_to_heads_kernel<X, D, VEC, 1, 1>;
  B200Q_CHECK_CUDA(launch_k(kernel, dim3(ceil_div(n_rows, rows), ceil_div(p.heads, block / TPH * std::max(it, 1))), dim3(block), 0, st, pdl, p, n_rows));
  return B200Q_OK;
}
template <typename X, int D>
int launch_dim(const RowsParams& p, int n_rows, bool vec, bool pdl, cudaStream_t st) {
  constexpr int VEC = 16 / (int)sizeof(X);
  return vec ? launch_vec<X, D, VEC>(p, n_rows, pdl, st) : launch_vec<X, D, 1>(p, n_rows, pdl, st);
}
template <typename X>
int launch_type(const RowsParams& p, int dim, int n_rows, bool vec, bool pdl, cudaStream_t st) {
  switch (dim) {
    case 16: return launch_dim<X, 16>(p, n_rows, vec, pdl, st);
    case 32: return launch_dim<X, 32>(p, n_rows, vec, pdl, st);
    case 64: return launch_dim<X, 64>(p, n_rows, vec, pdl, st);
    default: return launch_dim<X, 128>(p, n_rows, vec, pdl, st);
  }
}
// 16 bytes at a time where everything is on such boundaries: rows, outputs, and the halves of the rotated and of the other values
int launch_rows(const RowsParams& p, int x_dtype, int dim, int n_rows, bool pdl, cudaStream_t st) {
  const int xs = type_size(x_dtype), qs = type_size(p.q_dtype), vec = 16 / xs, half = p.rope ? p.rope_dim / 2 : 0;
  const bool wide = dim / 2 % vec == 0 && half % vec == 0 && (dim / 2 - half) % vec == 0 && !(((uintptr_t)p.x | (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v) & 15) &&
                    p.x_stride * xs % 16 == 0 && p.q_stride * qs % 16 == 0 && !((uintptr_t)p.rope & 15) && !(((uintptr_t)p.q_norm | (uintptr_t)p.k_norm) & (2 * vec - 1));
  if (x_dtype == B200Q_F32) return launch_type<float>(p, dim, n_rows, wide, pdl, st);
  if (x_dtype == B200Q_F16) return launch_type<__half>(p, dim, n_rows, wide, pdl, st);
  return launch_type<__nv_bfloat16>(p, dim, n_rows, wide, pdl, st);
}

int check_rotation(const float* rope, int rope_dim, int rope_len, int dim) {
  if (!rope) return B200Q_OK;
  if (rope_dim <= 0 || rope_len <= 0) return B200Q_ERR_BAD_ARG;
  if (rope_dim % 2 || rope_dim > dim) return B200Q_ERR_BAD_SHAPE;
  return (uintptr_t)rope & 3 ? B200Q_ERR_MISALIGNED : B200Q_OK;
}

}  // namespace

int b200q_paged_status_take(int* status) {
  int zero = 0;
  B200Q_CHECK_CUDA(cudaMemcpyFromSymbol(status, g_paged_status, sizeof(int)));
  B200Q_CHECK_CUDA(cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(int)));
  return B200Q_OK;
}

extern "C" int b200q_paged_append(const b200q_paged_cache* cache, const b200q_paged_batch* batch, const b200q_paged_append_args* a, int flags, void* stream) {
  int rc = check_cache(cache);
  if (rc == B200Q_OK) rc = check_batch(batch);
  if (rc != B200Q_OK) return rc;
  if (!a || a->n_heads <= 0 || !type_known(a->x_dtype) || !type_known(a->q_dtype)) return B200Q_ERR_BAD_ARG;
  const int dim = cache->head_dim;
  const int64_t q_row = (int64_t)a->n_heads * dim, row = q_row + 2 * (int64_t)cache->n_kv_heads * dim;
  if ((a->x_stride && a->x_stride < row) || (a->q_stride && a->q_stride < q_row) || row > INT32_MAX) return B200Q_ERR_BAD_SHAPE;
  if ((rc = check_rotation(a->rope, a->rope_dim, a->rope_len, dim)) != B200Q_OK) return rc;
  if (batch->n_seqs == 0 || batch->n_rows == 0) return B200Q_OK;
  if (!a->x || !a->q) return B200Q_ERR_BAD_ARG;
  if ((uintptr_t)a->x % type_size(a->x_dtype) || (uintptr_t)a->q % type_size(a->q_dtype) || ((uintptr_t)a->q_norm | (uintptr_t)a->k_norm) & 1) return B200Q_ERR_MISALIGNED;
  if (a->x == a->q && (a->x_dtype != a->q_dtype || (a->x_stride ? a->x_stride : row) != (a->q_stride ? a->q_stride : q_row))) return B200Q_ERR_BAD_ARG;      // rows would be overwritten before they are read
  const RowsParams p{a->x, a->q, cache->k, cache->v, a->q_dtype, cache->dtype, a->x_stride ? a->x_stride : row, a->q_stride ? a->q_stride : q_row, cache->page_stride,
                     cache->head_stride, cache->row_stride, a->n_heads, cache->n_kv_heads, a->n_heads + 2 * cache->n_kv_heads, a->norm_eps, (const __half*)a->q_norm,
                     (const __half*)a->k_norm, a->rope, a->rope_dim, a->rope_len, nullptr, divisor_of(cache->page_size), tables_of(cache, batch)};
  return launch_rows(p, a->x_dtype, dim, batch->n_rows, flags & B200Q_FLAG_PDL, (cudaStream_t)stream);
}

extern "C" int b200q_head_norm_rope(const b200q_head_norm_args* a, int flags, void* stream) {
  if (!a || a->n_rows < 0 || a->n_heads < 0 || a->n_kv_heads < 0 || a->n_heads + (int64_t)a->n_kv_heads <= 0 || !type_known(a->x_dtype) || !type_known(a->out_dtype)) return B200Q_ERR_BAD_ARG;
  if (a->head_dim != 16 && a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return B200Q_ERR_BAD_SHAPE;
  const int64_t row = ((int64_t)a->n_heads + a->n_kv_heads) * a->head_dim;
  if ((a->x_stride && a->x_stride < row) || (a->out_stride && a->out_stride < row) || row > INT32_MAX) return B200Q_ERR_BAD_SHAPE;
  const int rc = check_rotation(a->rope, a->rope_dim, a->rope_len, a->head_dim);
  if (rc != B200Q_OK) return rc;
  if (a->n_rows == 0) return B200Q_OK;
  if (!a->x || !a->out || (a->rope && !a->positions)) return B200Q_ERR_BAD_ARG;
  if ((uintptr_t)a->x % type_size(a->x_dtype) || (uintptr_t)a->out % type_size(a->out_dtype) || ((uintptr_t)a->q_norm | (uintptr_t)a->k_norm) & 1 || (uintptr_t)a->positions & 3) return B200Q_ERR_MISALIGNED;
  if (a->x == a->out && (a->x_dtype != a->out_dtype || (a->x_stride ? a->x_stride : row) != (a->out_stride ? a->out_stride : row))) return B200Q_ERR_BAD_ARG;
  const RowsParams p{a->x, a->out, nullptr, nullptr, a->out_dtype, 0, a->x_stride ? a->x_stride : row, a->out_stride ? a->out_stride : row, 0, 0, 0, a->n_heads,
                     a->n_kv_heads, a->n_heads + a->n_kv_heads, a->norm_eps, (const __half*)a->q_norm, (const __half*)a->k_norm, a->rope, a->rope_dim, a->rope_len,
                     a->positions, Divisor{}, PagedTables{}};
  return launch_rows(p, a->x_dtype, a->head_dim, a->n_rows, flags & B200Q_FLAG_PDL, (cudaStream_t)stream);
}
