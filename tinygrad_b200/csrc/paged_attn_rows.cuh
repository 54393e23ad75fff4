// Attention over pages for few rows (single tokens and short chunks): paged_attn.cu includes this.
//
// Bound by the keys and values, which are read once: 2 n_kv head_dim 2 bytes a position.  A tile is 16 (token, head) pairs, the rows of an m16n8k16 tensor-core instruction, so the work on
// a key is one instruction for all heads of its group.  Every warp streams blocks of 16 positions of its own through its own ring of asynchronous copies (no block-wide barrier
// until the end): 4 warps x 3 stages x 8 KB, two CTAs an SM, so that 128 KB are on their way in every SM while 64 KB are computed on (one microsecond of HBM's rate is 44 KB an SM).
//
// Precision: `N` 16-bit parts of a query and of a probability, each product a tensor-core pass of its own.  1 where queries, cache and output are all 16-bit: a probability loses half a step, as the
// output does; fp32 rows on fp16 keys 2 (2^-22; a row is scaled by a power of two that keeps it in fp16's range, probabilities by 2^14, which cancels in the quotient); on bf16 keys
// 3.  The tensor core cuts its sums where others round, so a block's weighted sum starts from zero and is added outside: with one running sum over 8192 positions the result is off by 1e-5.
#pragma once

namespace {

constexpr int RW = 4, R_THREADS = RW * 32, KB = 16;
template <int D> constexpr int R_BLOCK = KB * D * 2;                                      // bytes of a block's keys (or values)
template <int D> constexpr int R_STAGES = D == 128 ? 3 : D == 64 ? 6 : 8;
template <int D> constexpr int R_SMEM = RW * R_STAGES<D> * 2 * R_BLOCK<D> > RW * 16 * D * 4 ? RW * R_STAGES<D> * 2 * R_BLOCK<D> : RW * 16 * D * 4;

template <bool BF>
__device__ __forceinline__ void mma_row(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ float2 unpack2(uint32_t w, bool bf) {
  if (bf) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// a pair of values as N pairs of 16-bit values whose sum it is
template <int N, bool BF>
__device__ __forceinline__ void parts_of(float a, float b, uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    w[i] = pack2(a, b, BF ? B200Q_BF16 : B200Q_F16);
    if (i + 1 < N) { const float2 f = unpack2(w[i], BF); a -= f.x; b -= f.y; }
  }
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
// two 16-bit values, those that are infinite or NaN replaced by 0
template <bool BF> __device__ __forceinline__ uint32_t finite_only(uint32_t x) {
  constexpr uint32_t E = BF ? 0x7F80u : 0x7C00u;
  return ((x & E) == E ? 0u : x & 0xFFFFu) | ((x >> 16 & E) == E ? 0u : x & 0xFFFF0000u);
}
// 16-byte chunk c of row r of a block: the eight rows that an ldmatrix reads at once lie in different banks
template <int D> __device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  constexpr int CH = D / 8, SW = CH < 8 ? CH : 8;
  return r * (D * 2) + ((c ^ ((r / (8 / SW)) & (SW - 1))) << 4);
}
__device__ __forceinline__ float2 load2_as_f(const void* base, int type, int64_t i) {
  if (type == B200Q_F32) return make_float2(static_cast<const float*>(base)[i], static_cast<const float*>(base)[i + 1]);
  const uint16_t* p = static_cast<const uint16_t*>(base) + i;
  return unpack2(p[0] | (uint32_t)p[1] << 16, type == B200Q_BF16);
}

template <int D, int N, bool BF>
__global__ void __launch_bounds__(R_THREADS, 2) attn_rows_kernel(const AttnParams p) {
  constexpr int R = 16, CH = D / 8, ST = R_STAGES<D>, BLOCK = R_BLOCK<D>, KK = D / 16;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float s_m[RW][R], s_l[RW][R];
  __shared__ int s_flag;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3, kvh = blockIdx.y, split = blockIdx.z;
  const int ps = p.t.page_size, k_begin = split * p.split_len;
  const bool whole = ps % KB == 0;                      // a block lies in one page
  auto block_key = [&](int it) { return k_begin + (warp + it * RW) * KB; };
  // pages of this and the next 32 blocks; asked for before it is known how many of them there are, together with what says so
  auto page_id = [&](int seq, int it) {
    const int index = block_key(it) / ps;
    return whole && index < p.t.table_stride ? p.t.pages[(int64_t)seq * p.t.table_stride + index] : -1;
  };
  int ids = p.tiles_per_seq ? page_id(blockIdx.x / p.tiles_per_seq, lane) : 0;
  const TilePlace w = place_of_tile<R>(p, blockIdx.x);
  if (w.n == 0) return;
  const int n_parts = max(1, (w.keys + p.split_len - 1) / p.split_len), k_end = min(w.keys, k_begin + p.split_len);
  if (split >= n_parts) return;
  if (!p.tiles_per_seq) ids = page_id(w.seq, lane);
  const int pairs = w.n * p.group;
  const int blocks = max(0, (k_end - k_begin + KB - 1) / KB), mine = (blocks - warp + RW - 1) / RW;      // this warp's: warp, warp + RW, ...
  const uint16_t* kp = static_cast<const uint16_t*>(p.k) + kvh * p.head_stride;
  const uint16_t* vp = static_cast<const uint16_t*>(p.v) + kvh * p.head_stride;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(ring) + warp * (ST * 2 * BLOCK);
  int ids_next = mine > 32 ? page_id(w.seq, 32 + lane) : 0;
  auto issue = [&](int it) {
    if (it < mine) {
      const int key0 = block_key(it);
      const uint32_t to = base + (it % ST) * (2 * BLOCK);
      int64_t at0 = 0;
      bool there0 = true;
      if (whole) {
        const int page = __shfl_sync(0xffffffffu, ids, it & 31);
        if ((it & 31) == 31) { ids = ids_next; ids_next = mine > it + 33 ? page_id(w.seq, it + 33 + lane) : 0; }
        there0 = page >= 0 && page < p.t.n_pages;
        if (!there0 && lane == 0) atomicExch(&g_paged_attn_status, 2);
        at0 = there0 ? page * p.page_stride + (int64_t)(key0 % ps) * p.row_stride : 0;
      }
#pragma unroll
      for (int i = 0; i < (KB * CH + 31) / 32; i++) {
        const int c = lane + i * 32, r = c / CH, col = c % CH;
        bool there = there0 && key0 + r < k_end;
        int64_t at = at0 + (int64_t)r * p.row_stride;
        if (!whole) { at = there ? key_at(p, w.seq, key0 + r) : -1; there = at >= 0; }
        at = there ? at + col * 8 : 0;
        const uint32_t o = to + chunk_at<D>(r, col);
        copy16(o, kp + at, there ? 16 : 0);              // (nothing there: zeros)
        copy16(o + BLOCK, vp + at, there ? 16 : 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // the queries, as the instruction's A operand: rows g and g + 8.  All loads first (one that waits for the one before it is 5 us a CTA), then the first blocks, then the parts.
  float2 f[2][2 * KK];
  int last[2];                                           // the position a row may see up to
  {
    int64_t at[2];
    bool live[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int pair = w.r0 + g + e * 8, token = pair / p.group;
      live[e] = pair < pairs;
      last[e] = live[e] ? w.length + token : -1;
      at[e] = live[e] ? (w.first_row + token) * p.q_stride + (int64_t)(kvh * p.group + pair - token * p.group) * D + tq * 2 : 0;
    }
    const int size = type_size(p.q_dtype);
    const bool paired = (((uintptr_t)p.q | (uintptr_t)(p.q_stride * size)) & (2 * size - 1)) == 0;
    if (p.q_dtype == B200Q_F32 && paired) {
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int j = 0; j < 2 * KK; j++) f[e][j] = live[e] ? *reinterpret_cast<const float2*>(static_cast<const float*>(p.q) + at[e] + j * 8) : make_float2(0.f, 0.f);
    } else if (paired) {
      uint32_t x[2][2 * KK];
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int j = 0; j < 2 * KK; j++) x[e][j] = live[e] ? *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.q) + at[e] + j * 8) : 0u;
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int j = 0; j < 2 * KK; j++) f[e][j] = unpack2(x[e][j], p.q_dtype == B200Q_BF16);
    } else {
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int j = 0; j < 2 * KK; j++) f[e][j] = live[e] ? load2_as_f(p.q, p.q_dtype, at[e] + j * 8) : make_float2(0.f, 0.f);
    }
  }
#pragma unroll
  for (int i = 0; i < ST - 1; i++) issue(i);
  uint32_t qa[N][KK][4];
  float qs[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    float up = 1.f, down = 1.f;
    if (N == 2) {
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < 2 * KK; j++) amax = fmaxf(amax, fmaxf(fabsf(f[e][j].x), fabsf(f[e][j].y)));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      pow2_scale(amax, up, down);
    }
    qs[e] = p.scale * down;
#pragma unroll
    for (int j = 0; j < 2 * KK; j++) {
      uint32_t v[N];
      parts_of<N, BF>(f[e][j].x * up, f[e][j].y * up, v);
#pragma unroll
      for (int i = 0; i < N; i++) qa[i][j / 2][(j & 1) * 2 + e] = v[i];
    }
  }

  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < D / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  const int first_last = w.length + w.r0 / p.group;      // what the tile's first row sees: blocks up to it are seen by all
#pragma unroll 1
  for (int it = 0; it < mine; it++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
    __syncwarp();
    issue(it + ST - 1);
    const uint32_t ks = base + (it % ST) * (2 * BLOCK), vs = ks + BLOCK;
    const int key0 = block_key(it);
    float s[2][4] = {};
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
      uint32_t b[4];
      ldsm4(b, ks + chunk_at<D>((lane & 7) + (lane >> 4) * 8, kk * 2 + ((lane >> 3) & 1)));
#pragma unroll
      for (int i = N - 1; i >= 0; i--) { mma_row<BF>(s[0], qa[i][kk], b[0], b[1]); mma_row<BF>(s[1], qa[i][kk], b[2], b[3]); }
    }
    const bool masked = key0 + KB - 1 > first_last || key0 + KB > k_end;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int key = key0 + j * 8 + tq * 2 + (e & 1);
        s[j][e] *= qs[e >> 1];
        if (masked && (key > last[e >> 1] || key >= k_end)) s[j][e] = -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
      }
    float c[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
      mx[e] = fmaxf(mx[e], m[e]);
      c[e] = mx[e] == -INFINITY ? 1.f : exp2f(m[e] - mx[e]);
      m[e] = mx[e];
      l[e] *= c[e];
    }
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float sh = m[e >> 1] == -INFINITY ? 0.f : m[e >> 1] - 14.f;
        s[j][e] = exp2f(s[j][e] - sh);
        l[e >> 1] += s[j][e];
      }
    uint32_t pa[N][4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      uint32_t v[N];
      parts_of<N, BF>(s[e >> 1][(e & 1) * 2], s[e >> 1][(e & 1) * 2 + 1], v);
#pragma unroll
      for (int i = 0; i < N; i++) pa[i][e] = v[i];
    }
    bool odd = false;      // a value that is not finite, in a block that some rows do not see whole: 0 times it is not 0
    if (masked) {
      for (int i = lane; i < KB * CH; i += 32) {
        uint32_t x[4];
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(vs + i * 16) : "memory");
#pragma unroll
        for (int j = 0; j < 4; j++) odd |= finite_only<BF>(x[j]) != x[j];
      }
      odd = __any_sync(0xffffffffu, odd);
    }
#pragma unroll
    for (int n = 0; n < D / 16; n++) {
      uint32_t b[4];
      ldsm4_t(b, vs + chunk_at<D>((lane & 7) + ((lane >> 3) & 1) * 8, n * 2 + (lane >> 4)));
      if (odd) {
#pragma unroll
        for (int j = 0; j < 4; j++) b[j] = finite_only<BF>(b[j]);
      }
      float t[2][4] = {};
#pragma unroll
      for (int i = N - 1; i >= 0; i--) { mma_row<BF>(t[0], pa[i], b[0], b[1]); mma_row<BF>(t[1], pa[i], b[2], b[3]); }
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[2 * n + x][e] = fmaf(o[2 * n + x][e], c[e >> 1], t[x][e]);
    }
    if (odd) {             // what was left out, for the rows that see it (the others keep their bits)
#pragma unroll
      for (int j = 0; j < KB; j++) {
        float e2[2];
#pragma unroll
        for (int e = 0; e < 2; e++) e2[e] = __shfl_sync(0xffffffffu, s[j / 8][e * 2 + (j & 1)], (lane & ~3) | (j & 7) / 2);
        const bool sees[2] = {key0 + j <= last[0], key0 + j <= last[1]};
#pragma unroll
        for (int n = 0; n < D / 8; n++) {
          uint32_t x;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(vs + chunk_at<D>(j, n) + tq * 4) : "memory");
          const uint32_t left = x ^ finite_only<BF>(x);      // the values that are not finite, zeros elsewhere
          const float2 v = unpack2(left, BF);
#pragma unroll
          for (int e = 0; e < 2; e++) {
            if (sees[e] && (left & 0xFFFFu)) o[n][e * 2] = fmaf(e2[e], v.x, o[n][e * 2]);
            if (sees[e] && left >> 16) o[n][e * 2 + 1] = fmaf(e2[e], v.y, o[n][e * 2 + 1]);
          }
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // the warps' sums, in the order of the warps
#pragma unroll
  for (int e = 0; e < 2; e++) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    if (tq == 0) { s_m[warp][g + e * 8] = m[e]; s_l[warp][g + e * 8] = l[e]; }
  }
  __syncthreads();
  float* const s_o = reinterpret_cast<float*>(ring);       // [warp][R][D]
  float mt[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int r = g + e * 8;
    mt[e] = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    const float c = l[e] == 0.f ? 0.f : exp2f(m[e] - mt[e]);
#pragma unroll
    for (int n = 0; n < D / 8; n++) *reinterpret_cast<float2*>(s_o + (warp * R + r) * D + n * 8 + tq * 2) = make_float2(l[e] == 0.f ? 0.f : o[n][e * 2] * c, l[e] == 0.f ? 0.f : o[n][e * 2 + 1] * c);
  }
  __syncthreads();
  const int unit = blockIdx.x * p.n_kv + kvh;
  float* const part = p.parts + ((int64_t)unit * p.n_split + split) * PART<R, D>;
  for (int i = tid; i < R * D / 4; i += R_THREADS) {
    const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
    const int pair = w.r0 + r;
    if (pair >= pairs) break;
    float ml = -INFINITY, sum = 0.f, v[4] = {};
#pragma unroll
    for (int x = 0; x < RW; x++) ml = fmaxf(ml, s_m[x][r]);
#pragma unroll
    for (int x = 0; x < RW; x++) {
      const float lx = s_l[x][r];
      sum += lx == 0.f ? 0.f : lx * exp2f(s_m[x][r] - ml);
      const float4 f = *reinterpret_cast<const float4*>(s_o + (x * R + r) * D + d);
      v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
    }
    if (n_parts == 1) {
      const int token = pair / p.group;
      const int64_t at = (w.first_row + token) * p.out_stride + (int64_t)(kvh * p.group + pair - token * p.group) * D + d;
#pragma unroll
      for (int j = 0; j < 4; j++) store_as(p.out, p.out_dtype, at + j, sum == 0.f ? 0.f : v[j] / sum);
    } else {
      if (d == 0) { __stcg(part + r, ml); __stcg(part + R + r, sum); }
      __stcg(reinterpret_cast<float4*>(part + 2 * R + r * D + d), make_float4(v[0], v[1], v[2], v[3]));
    }
  }
  if (n_parts > 1) join_parts<R, D, R_THREADS>(p, w, unit, n_parts, kvh, &s_flag, s_o);
}

}  // namespace
