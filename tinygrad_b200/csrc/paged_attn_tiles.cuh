// Attention over pages for many rows (prompts and chunks): paged_attn.cu includes this.
//
// Bound by the tensor core and, as much, by what turns scores into probabilities: 256 rows x 128 keys are 2 x 256 x 128 x D multiply-adds (2048 cycles of the tensor core at D = 128), 32768 powers
// (2048 cycles of the special-function units) and some 600 instructions of each of the eight warps that see them.  So a CTA has two tiles of 128 rows whose products and softmaxes take turns: while one's
// scores are turned into probabilities, the other's products run.  Warps 0-3 and 4-7 are the tiles' softmax, a thread a row (scores are read from tensor memory as it holds them, no exchange between
// threads; two threads a row, half of its scores each, were slower); one thread issues the products, S = Q K^T from shared memory and O += P V with P from tensor memory; one warp brings keys, one values (TMA
// boxes of a page's rows, 128-byte swizzle), one looks after the values that a product must not see.  All powers are the special-function
// units': a quarter of them as a polynomial on the multiply-adders, whose results below 2^-126 have to be made 0, took 443 against 429 us below (heads of 64 312 against 302).  A tile's product begins with half of its probabilities.
//
// Tensor memory: S0 S1 O0 O1, 128 columns each, a tile's probabilities in the place of its scores.  Heads of 64 leave room for probabilities of their own (T_APART): the next scores
// are then computed as soon as these have been read, not behind their product (4096 rows of 32 heads of 64, 8192 positions: 302 us against 315 in place; 294 since the powers stand there once).
//
// 4096 rows of 32 heads of 128 at 8192 positions: 365 to 430 us, as the power limit has the clock (0.96 to 1.1 PFLOP/s).  CTAs that stay and share the work evenly took 442 against
// 388 us there, softmaxes that are kept apart by barriers 406 against 391, a running maximum looked for behind the first powers 399 against 388.
//
// The running maximum moves only when it has grown by 2^8: until then probabilities are relative to an older one, which the quotient does not notice, and the weighted sums
// in tensor memory stay as they are.
//
// Precision: N = 1, 16-bit queries and outputs: a probability loses half a step, as the output does.  N = 2, fp32 rows on fp16 keys: queries (under a power of two that keeps the row in range) and
// probabilities are two halves each, and a tile's weighted sum starts from zero and is added in registers, because the tensor core cuts its sums where others round.
#pragma once

namespace {

constexpr int T_ROWS = 128, T_R = 2 * T_ROWS, T_KEYS = 128, T_THREADS = 384, T_BASE = 7, T_PARTS = 16;      // probabilities up to 2^(7 + 8)
template <int D> constexpr int T_TILE = T_KEYS * D * 2;                                     // bytes of 128 rows of 16-bit values
template <int D, int N> constexpr int T_KS = D == 64 ? 3 : N == 1 ? 2 : 1;
template <int D, int N> constexpr bool T_APART = D == 64 && N == 1;      // probabilities have columns of their own
template <int D, int N> constexpr int T_VS = D == 64 ? 3 : N == 1 ? 3 : 2;
template <int D, int N> constexpr int T_SMEM = (2 * N + T_KS<D, N> + T_VS<D, N>) * T_TILE<D> + 1024;

struct SharedA {
  uint64_t k_full[3], k_empty[3], v_full[3], v_clean[3], v_empty[3], s_full[2], s_free[2], p_full[2][2], p_free[2], q_full, o_full;
  uint32_t tmem;
  int abort, flag, bad_lo, bad_hi;
};

__device__ __forceinline__ bool a_wait(SharedA& sh, uint64_t* b, uint32_t parity) { return bar_ready(b, parity) || a_wait_on(s_addr(b), parity, s_addr(&sh.abort)); }
__device__ __forceinline__ void a_commit(uint64_t* b) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s_addr(b)) : "memory"); }

// Operands in the 128-byte-swizzle layout: sub-tiles of 64 values (128 bytes) a row, 8 rows = 1024 bytes.  Q and K are read along a row (rows 1024 bytes per 8 apart); V, whose reduction runs over
// its rows, across them: then the distance between sub-tiles stands in the other field.
// A descriptor's low word (start, the other distance); the high one is the same for all.  Steps along an operand are added to the low word (16 bytes), so that the issuing thread has few values to keep.
constexpr uint32_t DESC_HI = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_128(uint32_t addr, uint32_t other) { return ((addr >> 4) & 0x3FFF) | (other >> 4) << 16; }
template <bool BF, bool ACROSS> __host__ __device__ constexpr uint32_t idesc_of(int n) {
  return 1u << 4 | (BF ? 1u << 7 | 1u << 10 : 0u) | (ACROSS ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(T_ROWS >> 4) << 24;
}
__device__ __forceinline__ void mma_ss_a(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n.reg .pred p;\n.reg .b64 x, y;\nmov.b64 x, {%1, %5};\nmov.b64 y, {%2, %5};\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}"
               ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(DESC_HI) : "memory");
}
__device__ __forceinline__ void mma_ts_a(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n.reg .pred p;\n.reg .b64 y;\nmov.b64 y, {%2, %5};\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}"
               ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(DESC_HI) : "memory");
}
__device__ __forceinline__ void ld32(uint32_t a, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
                 "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
                 "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]) : "r"(a));
}
__device__ __forceinline__ void st32(uint32_t a, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
               ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
                 "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
                 "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
}
__device__ __forceinline__ void ld16(uint32_t a, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
                 "=r"(v[14]), "=r"(v[15]) : "r"(a));
}
__device__ __forceinline__ void st8(uint32_t a, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void st16(uint32_t a, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
                 "r"(v[15]) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ uint4 ld_s4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

template <int V> struct Count { static constexpr int value = V; };
// two fp32 values at a time
__device__ __forceinline__ uint64_t pair_of(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float2 floats_of(uint64_t r) { float2 f; asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(r)); return f; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }      // NaN if one is

struct RowOf { int64_t row, head; int last; bool live; };      // of a thread: its row of the arrays, its head, the position it sees up to

// What a row that sees keys [lo, hi] with values that are not finite gets of them (their finite values are in the products already): added to its 32 columns from d0 on, which wait in shared memory.
template <bool BF>
__device__ __forceinline__ void add_not_finite(const AttnParams& p, int seq, int kvh, int lo, int hi, int d0, uint32_t row, int swizzle) {
#pragma unroll 1
  for (int key = lo; key <= hi; key++) {
    const int64_t at = key_at(p, seq, key);
    if (at < 0) continue;
    const uint16_t* v = static_cast<const uint16_t*>(p.v) + kvh * p.head_stride + at + d0;
#pragma unroll 1
    for (int d = 0; d < 32; d++) {
      const uint32_t x = v[d], a = row + (((d >> 2) ^ swizzle) << 4) + (d & 3) * 4;
      if (finite_only<BF>(x) == x) continue;
      float y;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(a) : "memory");
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(y + unpack2(x, BF).x) : "memory");
    }
  }
}

template <int D, int N, bool BF>
__global__ void __launch_bounds__(T_THREADS, 1) attn_tiles_kernel(const AttnParams p, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, int box_rows) {
  constexpr int SUBS = D / 64, TILE = T_TILE<D>, SUB = T_KEYS * 128, KS = T_KS<D, N>, VS = T_VS<D, N>, KK = D / 16;
  constexpr bool APART = T_APART<D, N>;
  constexpr int O_AT = 256, O_STEP = APART ? 64 : 128, P_AT = APART ? 384 : 0, P_STEP = APART ? 64 : 128, P_CHUNK = APART ? 16 : 32;      // columns of tensor memory
  extern __shared__ unsigned char raw[];
  __shared__ SharedA sh;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int order = p.by_kv.div(blockIdx.x), kvh = blockIdx.x - order * p.n_kv, split = blockIdx.y;
  const int tile_index = p.by_kv.div(gridDim.x) - 1 - order;      // long ones first
  const TilePlace w = place_of_tile<T_R>(p, tile_index);
  const int n_parts = w.n == 0 ? 0 : parts_of_keys(p, w.keys), k_begin = split * p.split_len, k_end = k_begin + min(w.keys - k_begin, p.split_len);
  if (split >= n_parts) return;
  const int tiles = max(0, (k_end - k_begin + T_KEYS - 1) / T_KEYS);
  const int pairs = w.n * p.group;
  const bool two = w.r0 + T_ROWS < pairs;                      // the second tile of rows has some
  const int first_last = w.length + p.by_group.div(w.r0);            // what the first row sees
  const uint32_t s_q = (s_addr(raw) + 1023) & ~1023u, s_k = s_q + 2 * N * TILE, s_v = s_k + KS * TILE;

  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&sh.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < 3; i++) {
      a_bar_init(&sh.k_full[i], 1); a_bar_init(&sh.k_empty[i], 1); a_bar_init(&sh.v_full[i], 1); a_bar_init(&sh.v_clean[i], 1); a_bar_init(&sh.v_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) { a_bar_init(&sh.s_full[i], 1); a_bar_init(&sh.s_free[i], 4); a_bar_init(&sh.p_free[i], 1); a_bar_init(&sh.p_full[i][0], 4); a_bar_init(&sh.p_full[i][1], 4); }
    a_bar_init(&sh.q_full, 8); a_bar_init(&sh.o_full, 1);
    sh.abort = sh.flag = 0; sh.bad_lo = INT32_MAX; sh.bad_hi = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  const int unit = tile_index * p.n_kv + kvh;

  // registers: 384 threads x 168 = 64512 at launch = 256 x 208 + 128 x 88
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax: a thread a row ----
    const int t = warp >> 2, r = tid & 127;
    RowOf me;
    {
      const int pair = w.r0 + t * T_ROWS + r;
      me.live = pair < pairs;
      const int token = me.live ? p.by_group.div(pair) : 0;
      me.row = w.first_row + token;
      me.head = kvh * p.group + (me.live ? pair - token * p.group : 0);
      me.last = me.live ? w.length + token : -1;
    }
    float qs = p.scale;
    if (t == 0 || two) {
      // the warp's 32 rows of queries, whole rows at a time: N parts, chunks of 16 bytes in the swizzled places.  PER values a lane.
      constexpr int PER = N == 1 ? 8 : 4, LANES = D / PER, AT_ONCE = 32 / LANES;
      const int size = type_size(p.q_dtype), l = lane % LANES;
      const bool wide = (((uintptr_t)p.q | (uintptr_t)(p.q_stride * size)) & 15) == 0;
      auto row_at = [&](int i) {      // where this lane's values of the i-th run of rows are; -1: no row
        const int pair = w.r0 + t * T_ROWS + (warp & 3) * 32 + i * AT_ONCE + lane / LANES, token = p.by_group.div(pair);
        return pair < pairs ? (w.first_row + token) * p.q_stride + (int64_t)(kvh * p.group + pair - token * p.group) * D + l * PER : (int64_t)-1;
      };
      auto place = [&](int i, int part) {      // and where they go
        const int row = (warp & 3) * 32 + i * AT_ONCE + lane / LANES, chunk = l * PER / 8;
        return s_q + (part * 2 + t) * TILE + (chunk >> 3) * SUB + row * 128 + (((chunk & 7) ^ (row & 7)) << 4) + (PER == 4 ? (l & 1) * 8 : 0);
      };
      if constexpr (N == 1) {
        constexpr int RUNS = 32 / AT_ONCE;
        if (wide) {
          uint4 v[RUNS];
#pragma unroll
          for (int i = 0; i < RUNS; i++) {
            const int64_t at = row_at(i);
            v[i] = at >= 0 ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + at) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < RUNS; i++) st_s4(place(i, 0), v[i]);
        } else {
#pragma unroll 1
          for (int i = 0; i < RUNS; i++) {
            const int64_t at = row_at(i);
            uint32_t x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = at >= 0 ? pack2(load_as_f(p.q, p.q_dtype, at + 2 * j), load_as_f(p.q, p.q_dtype, at + 2 * j + 1), BF ? B200Q_BF16 : B200Q_F16) : 0u;
            st_s4(place(i, 0), make_uint4(x[0], x[1], x[2], x[3]));
          }
        }
      } else {
        float mine = 1.f;      // what undoes this thread's row's scaling
#pragma unroll 1
        for (int i0 = 0; i0 < 32 / AT_ONCE; i0 += 8) {
          float4 v[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int64_t at = row_at(i0 + i);
            v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at >= 0) {
              if (wide && p.q_dtype == B200Q_F32) v[i] = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at);
              else v[i] = make_float4(load_as_f(p.q, p.q_dtype, at), load_as_f(p.q, p.q_dtype, at + 1), load_as_f(p.q, p.q_dtype, at + 2), load_as_f(p.q, p.q_dtype, at + 3));
            }
          }
#pragma unroll
          for (int i = 0; i < 8; i++) {
            float amax = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w))), up, down;
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            pow2_scale(amax, up, down);
            if (amax == 0.f) down = 1.f;
            const float d = __shfl_sync(0xffffffffu, down, lane % AT_ONCE * LANES);
            if (lane / AT_ONCE == i0 + i) mine = d;
            uint32_t x[N], y[N];
            parts_of<N, BF>(v[i].x * up, v[i].y * up, x);
            parts_of<N, BF>(v[i].z * up, v[i].w * up, y);
#pragma unroll
            for (int q = 0; q < N; q++) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(place(i0 + i, q)), "r"(x[q]), "r"(y[q]) : "memory");
          }
        }
        qs *= mine;
      }
      qs = fmaxf(qs, 1.1754944e-38f);
    }
    fence_async();
    __syncwarp();
    if (lane == 0) a_bar_arrive(&sh.q_full);
    float m = -INFINITY, l = 0.f;
    [[maybe_unused]] float acc[N == 2 ? D : 1];
    if constexpr (N == 2) {
#pragma unroll
      for (int d = 0; d < D; d++) acc[d] = 0.f;
    }
    const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * 128, to = ts + O_AT - t * (128 - O_STEP), tp = ts + P_AT - t * (128 - P_STEP);
    const int warp_first = __shfl_sync(0xffffffffu, me.last, 0);      // no row of the warp sees less (rows without a token see nothing, and are not stored)
    bool ok = t == 0 || two;
    float scaled = 1.f;      // N == 2: what the sum in registers is multiplied by before a tile's is added
#pragma unroll 1
    for (int j = 0; ok && j < tiles; j++) {
      const int k0 = k_begin + j * T_KEYS;
      ok = __all_sync(0xffffffffu, a_wait(sh, &sh.s_full[t], j & 1));
      if (!ok) break;
      fence_after();
      const bool masked = k0 + T_KEYS - 1 > warp_first || k0 + T_KEYS > k_end;
      const int lim = min(me.last, k_end - 1) - k0;
      float top = -INFINITY;
      if constexpr (N == 1) {
        float s[128];
#pragma unroll
        for (int c = 0; c < 4; c++) ld32(ts + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
        wait_ld();
        if constexpr (APART) {
          fence_before();
          __syncwarp();
          if (lane == 0) a_bar_arrive(&sh.s_free[t]);
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 128; i++) s[i] = i <= lim ? s[i] : -INFINITY;
        }
        float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < 124; i += 8) {
#pragma unroll
          for (int q = 0; q < 4; q++) tops[q] = max3(tops[q], s[i + q], s[i + 4 + q]);
        }
#pragma unroll
        for (int q = 0; q < 4; q++) tops[q] = max3(tops[q], s[124 + q], s[124 + q]);
        top = max3(tops[0], tops[1], max3(tops[2], tops[3], tops[3])) * qs;
        if (!(top < INFINITY)) { l = __uint_as_float(0x7FC00000u); top = m; }      // a score that is infinite or NaN: the row is NaN, whatever takes its exponentials
        if constexpr (APART) {      // the product of the tile before has its probabilities, and its sum is there
          if (j > 0) ok = __all_sync(0xffffffffu, a_wait(sh, &sh.p_free[t], (j - 1) & 1));
          if (!ok) break;
          fence_after();
        }
        const bool moves = j == 0 || top > m + 8.f;
        if (__any_sync(0xffffffffu, moves)) {
          const float mn = fmaxf(m, top), f = mn == -INFINITY ? 1.f : pow2(m - mn);
          m = mn;
          if (j > 0) {
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
              uint32_t o[32];
              ld32(to + c * 32, o);
              wait_ld();
#pragma unroll
              for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              st32(to + c * 32, o);
            }
          }
        }
        const float sub = m == -INFINITY ? 0.f : T_BASE - m;
        const uint64_t qs2 = pair_of(qs, qs), sub2 = pair_of(sub, sub);
        uint64_t sums[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 4; c++) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const float2 x = floats_of(fma2(pair_of(s[c * 32 + 2 * i], s[c * 32 + 2 * i + 1]), qs2, sub2));
            const float a = pow2(x.x), b = pow2(x.y);      // (of minus infinity: 0, so that a row without a finite score ends with a sum of 0)
            sums[i & 1] = add2(sums[i & 1], pair_of(a, b));
            pk[i] = pack2(a, b, BF ? B200Q_BF16 : B200Q_F16);
          }
          st16(tp + c * P_CHUNK, pk);
          if (c & 1) {      // half of the tile's probabilities: the product begins with them
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) a_bar_arrive(&sh.p_full[t][c / 2]);
          }
        }
        const float2 y0 = floats_of(sums[0]), y1 = floats_of(sums[1]);
        l += (y0.x + y0.y) + (y1.x + y1.y);
      } else {
        // the tile before: its weighted sum is complete (the scores behind it in the tensor core's queue are)
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < D / 16; c++) {
            uint32_t o[16];
            ld16(to + c * 16, o);
            wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) acc[c * 16 + i] = fmaf(acc[c * 16 + i], scaled, __uint_as_float(o[i]));
          }
        }
#pragma unroll 1
        for (int c = 0; c < 4; c++) {
          float s[32];
          ld32(ts + c * 32, reinterpret_cast<uint32_t*>(s));
          wait_ld();
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; i++) s[i] = c * 32 + i <= lim ? s[i] : -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) top = max3(top, s[i], s[i + 1]);
        }
        top *= qs;
        if (!(top < INFINITY)) { l = __uint_as_float(0x7FC00000u); top = m; }
        const float mn = fmaxf(m, top);
        scaled = mn == -INFINITY ? 1.f : pow2(m - mn);
        m = mn;
        l *= scaled;
        const float sub = m == -INFINITY ? 0.f : T_BASE + 7 - m;
        float sum = 0.f;
#pragma unroll 2
        for (int c = 0; c < 8; c++) {                      // 16 keys: their high parts, then the low ones (8 columns each); half of the tile is handed over as soon as it is there
          float s[16];
          uint32_t hi[8], lo[8];
          ld16(ts + c * 16, reinterpret_cast<uint32_t*>(s));
          wait_ld();
          if (masked) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = c * 16 + i <= lim ? s[i] : -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float a = pow2(fmaf(s[2 * i], qs, sub)), b = pow2(fmaf(s[2 * i + 1], qs, sub));
            sum += a + b;
            uint32_t x[N];
            parts_of<N, BF>(a, b, x);
            hi[i] = x[0];
            lo[i] = x[N - 1];
          }
          st8(ts + c * 16, hi);
          st8(ts + c * 16 + 8, lo);
          if (c & 3 ^ 3) continue;
          wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) a_bar_arrive(&sh.p_full[t][c >> 2]);
        }
        l += sum;
      }
    }
    if (ok && tiles) ok = __all_sync(0xffffffffu, a_wait(sh, &sh.o_full, 0));
    // ---- what comes out ----
    if (ok) {
      fence_after();
      const int bad_lo = *(volatile int*)&sh.bad_lo, bad_hi = min(*(volatile int*)&sh.bad_hi, me.last);
      float* part = p.parts + ((int64_t)unit * p.n_split + split) * PART<T_R, D>;
      const int pr = t * T_ROWS + r;
      if (n_parts > 1 && me.live) { __stcg(part + pr, m); __stcg(part + T_R + pr, l); }
      const float inv = n_parts > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      const int64_t at = me.row * p.out_stride + me.head * D;
      const bool words = n_parts > 1 || p.out_dtype == B200Q_F32;      // 32-bit values leave
      const bool wide = n_parts > 1 || (((uintptr_t)p.out | (uintptr_t)(p.out_stride * (words ? 4 : 2))) & 15) == 0;
      const unsigned live = __ballot_sync(0xffffffffu, me.live);
      if constexpr (N == 2) {      // all of it in tensor memory, as of N == 1
#pragma unroll
        for (int c = 0; c < D / 16; c++) {
          uint32_t x[16];
          if (tiles) {
            ld16(to + c * 16, x);
            wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = __float_as_uint(fmaf(acc[c * 16 + i], scaled, __uint_as_float(x[i])));
            st16(to + c * 16, x);
          }
        }
        wait_st();
      }
      // 32 columns at a time through the place of the warp's queries, so that a store writes whole pieces of rows.  (Short loops: this runs once a CTA, and unrolled it took 12000 cycles, which its
      // instructions needed to come.)
      const uint32_t stage = s_q + t * TILE + (warp & 3) * (32 * 128);
      const float factor = l == 0.f ? 0.f : inv;
#pragma unroll 1
      for (int c = 0; c < D / 32; c++) {
        uint32_t x[32];
        if (tiles) { ld32(to + c * 32, x); wait_ld(); }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (tiles && l != 0.f) v = make_float4(__uint_as_float(x[i]) * factor, __uint_as_float(x[i + 1]) * factor, __uint_as_float(x[i + 2]) * factor, __uint_as_float(x[i + 3]) * factor);
          st_s4(stage + lane * 128 + (((i >> 2) ^ (lane & 7)) << 4), make_uint4(__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w)));
        }
        if (bad_lo <= bad_hi && me.live) add_not_finite<BF>(p, w.seq, kvh, bad_lo, bad_hi, c * 32, stage + lane * 128, lane & 7);
        __syncwarp();
        // PER_ROW lanes a row; body(row, its place in the outputs)
        auto rows = [&](auto lanes, auto body) {
          constexpr int PER_ROW = lanes.value;
#pragma unroll
          for (int i = 0; i < PER_ROW; i++) {
            const int row = i * (32 / PER_ROW) + lane / PER_ROW;
            const int64_t to_row = __shfl_sync(0xffffffffu, at, row) + c * 32;
            if (live >> row & 1) body(row, to_row);
          }
        };
        auto quad = [&](int row, int q) { return ld_s4(stage + row * 128 + ((q ^ (row & 7)) << 4)); };
        if (n_parts > 1)
          rows(Count<8>{}, [&](int row, int64_t) { __stcg(reinterpret_cast<uint4*>(part + 2 * T_R + (t * T_ROWS + (warp & 3) * 32 + row) * D + c * 32 + (lane & 7) * 4), quad(row, lane & 7)); });
        else if (wide && !words)
          rows(Count<4>{}, [&](int row, int64_t to_row) {
            const uint4 x = quad(row, (lane & 3) * 2), y = quad(row, (lane & 3) * 2 + 1);
            auto two_of = [&](uint32_t u, uint32_t v) { return pack2(__uint_as_float(u), __uint_as_float(v), p.out_dtype); };
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + to_row + (lane & 3) * 8) = make_uint4(two_of(x.x, x.y), two_of(x.z, x.w), two_of(y.x, y.y), two_of(y.z, y.w));
          });
        else if (wide)
          rows(Count<8>{}, [&](int row, int64_t to_row) { *reinterpret_cast<uint4*>(static_cast<float*>(p.out) + to_row + (lane & 7) * 4) = quad(row, lane & 7); });
        else
#pragma unroll 1
          for (int row = 0; row < 32; row++) {
            const int64_t to_row = __shfl_sync(0xffffffffu, at, row) + c * 32;
            float y;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(stage + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4) : "memory");
            if (live >> row & 1) store_as(p.out, p.out_dtype, to_row + lane, y);
          }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8) {
    // ---- products ----
    if (elect_one()) {
      constexpr uint32_t ID_S = idesc_of<BF, false>(T_KEYS), ID_O = idesc_of<BF, true>(D);
      const uint32_t q0 = desc_128(s_q, 16), k0 = desc_128(s_k, 16), v0 = desc_128(s_v, SUB);
      auto scores = [&](int t, int ks) {
        const uint32_t q = q0 + t * (TILE >> 4), k = k0 + ks * (TILE >> 4);
#pragma unroll
        for (int i = N - 1; i >= 0; i--)
#pragma unroll
          for (int kk = 0; kk < KK; kk++) {
            const uint32_t o = ((kk / 4) * SUB + (kk % 4) * 32) >> 4;
            mma_ss_a(tmem + t * 128, q + i * (2 * TILE >> 4) + o, k + o, ID_S, i < N - 1 || kk > 0);
          }
        a_commit(&sh.s_full[t]);
      };
      bool ok = tiles > 0 && a_wait(sh, &sh.q_full, 0) && a_wait(sh, &sh.k_full[0], 0);
      if (ok) {
        fence_after();
        scores(0, 0);
        if (two) scores(1, 0);
        a_commit(&sh.k_empty[0]);
      }
      for (int j = 0; ok && j < tiles; j++) {
        const int vs = j % VS, kn = (j + 1) % KS;
        const uint32_t v = v0 + vs * (TILE >> 4);
        if constexpr (!APART) ok = a_wait(sh, &sh.v_clean[vs], (j / VS) & 1);
        for (int t = 0; ok && t < 1 + two; t++) {
          if constexpr (APART) {      // the next scores as soon as these have been read
            if (j + 1 < tiles) {
              ok = (t == 1 || a_wait(sh, &sh.k_full[kn], ((j + 1) / KS) & 1)) && a_wait(sh, &sh.s_free[t], j & 1);
              if (!ok) break;
              fence_after();
              scores(t, kn);
              if (t == two) a_commit(&sh.k_empty[kn]);
            }
            if (t == 0) ok = a_wait(sh, &sh.v_clean[vs], (j / VS) & 1);
          }
          // the probabilities come in two halves; their small parts first
#pragma unroll
          for (int h = 0; h < 2; h++) {
            ok = ok && a_wait(sh, &sh.p_full[t][h], j & 1);
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int i = N - 1; i >= 0; i--)
#pragma unroll
              for (int kk = h * 4; kk < h * 4 + 4; kk++)
                mma_ts_a(tmem + O_AT + t * O_STEP, tmem + P_AT + t * P_STEP + (N == 1 ? (kk / 2) * P_CHUNK + (kk & 1) * 8 : kk * 16 + i * 8), v + kk * (2048 >> 4), ID_O,
                         h > 0 || i < N - 1 || kk > 0 || (N == 1 && j > 0));
          }
          if (!ok) break;
          if (t == two) a_commit(&sh.v_empty[vs]);
          if constexpr (APART) a_commit(&sh.p_free[t]);
          else if (j + 1 < tiles) {
            if (t == 0) { ok = a_wait(sh, &sh.k_full[kn], ((j + 1) / KS) & 1); if (!ok) break; fence_after(); }
            scores(t, kn);
            if (t == two) a_commit(&sh.k_empty[kn]);
          }
        }
      }
      a_commit(&sh.o_full);
      if (!ok) a_wait_on(s_addr(&sh.o_full), 0, s_addr(&sh.flag));      // products in flight are done before tensor memory goes back (flag is 0 here)
    }
  } else if (warp < 11) {
    // ---- keys (one warp), values (another): a lane a box ----
    const bool v = warp == 10;
    const int stages = v ? VS : KS, per_tile = T_KEYS / box_rows, ps = p.t.page_size, sub = lane % SUBS, pg = lane / SUBS;
    const uint32_t to = (v ? s_v : s_k) + sub * SUB + pg * box_rows * 128;
    uint64_t* const full = v ? sh.v_full : sh.k_full;
    uint64_t* const empty = v ? sh.v_empty : sh.k_empty;
    const int32_t* row_pages = p.t.pages + (int64_t)w.seq * p.t.table_stride;
    auto page_of = [&](int j) {
      const int key = k_begin + j * T_KEYS + pg * box_rows;
      return j < tiles && key < k_end && pg < per_tile ? row_pages[p.by_page.div(key)] : -1;
    };
    bool ok = true;
    int st = 0, use = 0, j = 0, next = page_of(0);
    for (; j < tiles; j++) {
      const int k0 = k_begin + j * T_KEYS, n_pages = min(per_tile, (k_end - k0 + box_rows - 1) / box_rows), slot = k0 + pg * box_rows - p.by_page.div(k0 + pg * box_rows) * ps;
      const bool mine = pg < n_pages;
      int page = next;
      next = page_of(j + 1);
      if (mine && (page < 0 || page >= p.t.n_pages)) { page = p.t.n_pages; atomicExch(&g_paged_attn_status, 2); }      // (outside the map: the box is filled with zeros)
      if (use > 0) ok = a_wait(sh, &empty[st], (use - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(s_addr(&full[st])), "r"(n_pages * SUBS * box_rows * 128) : "memory");
      __syncwarp();
      if (mine)
        asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                     ::"r"(to + st * TILE), "l"(v ? &tm_v : &tm_k), "r"(s_addr(&full[st])), "r"(sub * 64), "r"(slot), "r"(kvh), "r"(page) : "memory");
      __syncwarp();
      if (++st == stages) { st = 0; use++; }
    }
    if (!ok)        // copies in flight end before the shared memory does
      for (int x = max(0, j - stages); x < j; x++) a_wait_on(s_addr(&full[x % stages]), (x / stages) & 1, s_addr(&sh.flag));
  } else {
    // ---- values that a product must not see: rows behind the last key, and what is not finite in rows that not every query sees (0 times it is not 0) ----
    bool ok = true;
    int st = 0, use = 0;
    for (int j = 0; j < tiles; j++) {
      const int k0 = k_begin + j * T_KEYS;
      ok = __all_sync(0xffffffffu, a_wait(sh, &sh.v_full[st], use & 1));
      if (!ok) break;
      const int from = max(0, min(first_last + 1, k_end) - k0), behind = max(0, min(T_KEYS, k_end - k0));      // the first row that somebody does not see, that nobody sees
      if (from < T_KEYS) {
        // (Looking must be quick: the tile's product waits for it, and where it was not, the last product of a CTA came 8000 cycles late.  A value is not finite where its exponent and one more overflow.)
        constexpr uint32_t E = BF ? 0x7F807F80u : 0x7C007C00u, ONE = BF ? 0x00800080u : 0x04000400u;
        uint32_t odd = 0;
#pragma unroll 8
        for (int i = from * 8 + lane; i < behind * 8; i += 32) {
#pragma unroll
          for (int s = 0; s < SUBS; s++) {
            const uint4 x = ld_s4(s_v + st * TILE + s * SUB + i * 16);
            odd |= ((x.x & E) + ONE) | ((x.y & E) + ONE) | ((x.z & E) + ONE) | ((x.w & E) + ONE);
          }
        }
        bool changed = false;
        if (odd & 0x80008000u) {
#pragma unroll 1
          for (int i = from * 8 + lane; i < behind * 8; i += 32) {
#pragma unroll 1
            for (int s = 0; s < SUBS; s++) {
              const uint32_t a = s_v + st * TILE + s * SUB + i * 16;
              const uint4 x = ld_s4(a), y = make_uint4(finite_only<BF>(x.x), finite_only<BF>(x.y), finite_only<BF>(x.z), finite_only<BF>(x.w));
              if (x.x == y.x && x.y == y.y && x.z == y.z && x.w == y.w) continue;
              st_s4(a, y);
              changed = true;
              atomicMin(&sh.bad_lo, k0 + i / 8);
              atomicMax(&sh.bad_hi, k0 + i / 8);
            }
          }
        }
        for (int i = behind * 8 + lane; i < T_KEYS * 8; i += 32) {
#pragma unroll
          for (int s = 0; s < SUBS; s++) st_s4(s_v + st * TILE + s * SUB + i * 16, make_uint4(0, 0, 0, 0));
          changed = true;
        }
        if (changed) fence_async();
      }
      __syncwarp();
      if (lane == 0) a_bar_arrive(&sh.v_clean[st]);
      if (++st == VS) { st = 0; use++; }
    }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// The parts of tiles whose keys are split, added in the order of the keys: J_SLICES CTAs for a (tile, KV head); a warp a row, a lane a part for the parts' shares and D / 32 values for the sum.
constexpr int J_SLICES = 8, J_THREADS = 256;
static_assert(T_PARTS <= 32, "a lane a part");
template <int D>
__global__ void __launch_bounds__(J_THREADS) join_tiles_kernel(const AttnParams p) {
  constexpr int V = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int order = p.by_kv.div(blockIdx.x), kvh = blockIdx.x - order * p.n_kv, tile_index = p.by_kv.div(gridDim.x) - 1 - order, lane = threadIdx.x & 31;
  const TilePlace w = place_of_tile<T_R>(p, tile_index);
  const int n_parts = parts_of_keys(p, w.keys), end = min(T_R, w.n * p.group - w.r0);
  if (w.n == 0 || n_parts <= 1) return;
  const float* first = p.parts + (int64_t)(tile_index * p.n_kv + kvh) * p.n_split * PART<T_R, D>;
#pragma unroll 1
  for (int r = blockIdx.y * (J_THREADS / 32) + (threadIdx.x >> 5); r < end; r += J_SLICES * (J_THREADS / 32)) {
    float m = -INFINITY, l = 0.f, o[V] = {};
    if (lane < n_parts) { m = __ldcg(first + lane * PART<T_R, D> + r); l = __ldcg(first + lane * PART<T_R, D> + T_R + r); }
    const float top = warp_max(m), f = l == 0.f ? 0.f : pow2(m - top), sum = warp_sum(f * l);      // (a part without keys has sum 0)
#pragma unroll 4
    for (int q = 0; q < n_parts; q++) {
      const float* b = first + q * PART<T_R, D> + 2 * T_R + r * D + lane * V;
      const float g = __shfl_sync(0xffffffffu, f, q);
      float v[V];
      if constexpr (V == 4) { const float4 y = __ldcg(reinterpret_cast<const float4*>(b)); v[0] = y.x; v[1] = y.y; v[2] = y.z; v[3] = y.w; }
      else { const float2 y = __ldcg(reinterpret_cast<const float2*>(b)); v[0] = y.x; v[1] = y.y; }
#pragma unroll
      for (int i = 0; i < V; i++) o[i] = fmaf(g, v[i], o[i]);
    }
    const int pair = w.r0 + r, token = p.by_group.div(pair);
    const int64_t at = (w.first_row + token) * p.out_stride + (int64_t)(kvh * p.group + pair - token * p.group) * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; i++) store_as(p.out, p.out_dtype, at + i, sum == 0.f ? 0.f : o[i] / sum);
  }
}

}  // namespace
