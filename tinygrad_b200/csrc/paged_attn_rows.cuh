// Attention over pages for few rows (single tokens and short chunks): paged_attn.cu includes this.
//
// Bound by the keys and values, which are read once: 2 n_kv head_dim 2 bytes a position.  A tile is 16 (token, head) pairs, the rows of an m16n8k16 tensor-core instruction, so the work on
// a key is one instruction for all heads of its group.  Every warp streams blocks of 16 positions of its own through its own ring (no block-wide barrier until the end): 4 warps x 3 stages x 8 KB,
// two CTAs an SM, so that 128 KB are on their way in every SM while 64 KB are computed on (one microsecond of HBM's rate is 44 KB an SM).  A block comes as TMA boxes of its page, 64 values x 16
// positions in the 128-byte-swizzle layout; where pages or heads are no such boxes (page sizes that 16 does not divide, heads of 16 or 32), as 16-byte copies of the
// warp's lanes, which cost more instructions than all of the arithmetic (131071 positions: 115 us).
//
// The deal: all rounds of 64 positions of all (tile, KV head) units, in order, are cut into as many equal shares as there are CTAs, whatever the sequences' lengths.  A CTA goes through the units
// of its share one after the other; a unit that is cut leaves parts (a CTA has two places for them: that of a unit which began before its share and that of one which goes on behind it), which the CTA
// that is done last joins.
//
// Precision: `N` 16-bit parts of a query and of a probability, each product a tensor-core pass of its own.  1 where queries, cache and output are all 16-bit: a probability loses half a step, as the
// output does; fp32 rows on fp16 keys 2 (2^-22; a row is scaled by a power of two that keeps it in fp16's range, probabilities by 2^14, which cancels in the quotient); on bf16 keys
// 3.  The tensor core cuts its sums where others round, so a block's weighted sum starts from zero and is added outside: with one running sum over 8192 positions the result is off by 1e-5.
#pragma once
#include <cuda.h>
#include <string.h>

namespace {

constexpr int RW = 4, R_THREADS = RW * 32, KB = 16;
template <int D> constexpr int R_BLOCK = KB * D * 2;                                      // bytes of a block's keys (or values)
template <int D> constexpr int R_STAGES = D == 128 ? 3 : D == 64 ? 6 : 8;
template <int D> constexpr int R_RING = RW * R_STAGES<D> * 2 * R_BLOCK<D> > RW * 16 * D * 4 ? RW * R_STAGES<D> * 2 * R_BLOCK<D> : RW * 16 * D * 4;
// ROUND: positions of a round.  R_LEAST: rounds that a CTA has at least, where there are enough for an SM each.  R_LONG: rounds of a share from which the beginning and end of a unit count as R_EXTRA
// rounds.  us with 4 KV heads of 7 x 128, sequences of one new token, at 64 x 1000 / 32 x 1000 / 64 x 200 / 16 x 1000 / 3 x 8000 positions at most: R_LONG 12, R_LEAST 4 44.1 / 26.9 / 24.9 / 22.8 / 20.7 (units cut
// wherever a share ends, each in its two parts); R_LONG 2 27.7 / 20.7 / 22.2 / 18.7 / 20.7; R_LEAST 2 with it 27.6 / 18.8 / 18.7 / 16.7 / 22.8.  R_EXTRA 3 to 5 within 3 % of one another, 8: 31.0 / 22.8.
constexpr int ROUND = RW * KB, R_LEAST = 2;
constexpr uint32_t R_LONG = 2, R_EXTRA = 4;

__device__ __forceinline__ uint32_t s_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void a_bar_init(uint64_t* b, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s_addr(b)), "r"(n) : "memory"); }
__device__ __forceinline__ void a_bar_arrive(uint64_t* b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s_addr(b)) : "memory"); }
__device__ __forceinline__ bool bar_ready(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(s_addr(b)), "r"(parity) : "memory");
  return ok;
}
// Bounded wait: false when the time is over (then the others are told), or once another has given up and a little longer has not helped: what was in flight has had its time before
// anything else happens to its place, or the kernel ends.
__device__ __forceinline__ bool a_wait_on(uint32_t bar, uint32_t parity, uint32_t abort) {
  for (int i = 0; i < (1 << 20); i++) {
    uint32_t ok, gone;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity), "r"(2000) : "memory");
    if (ok) return true;
    asm volatile("ld.volatile.shared::cta.u32 %0, [%1];" : "=r"(gone) : "r"(abort) : "memory");
    if (gone && i >= 1000) return false;
  }
  asm volatile("st.volatile.shared::cta.u32 [%0], 1;" ::"r"(abort) : "memory");
  atomicExch(&g_paged_attn_status, 1);
  return false;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float pow2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void st_s4(uint32_t a, uint4 v) { asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }

template <bool BF>
__device__ __forceinline__ void mma_row(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF>      // the same on sums that start from zero
__device__ __forceinline__ void mma_row0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
// 16-byte chunk c of row r of a block: the eight rows that an ldmatrix reads at once lie in different banks.  Heads of 64 and more: sub-blocks of 64 values, as the boxes leave them.
template <int D> constexpr int ROW_BYTES = D >= 64 ? 128 : D * 2;
template <int D> __device__ __forceinline__ uint32_t row_swizzle(int r) { return D >= 64 ? r & 7 : D == 32 ? (r >> 1) & 3 : (r >> 2) & 1; }
template <int D> __device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (c >> 3) * (KB * 128) + r * ROW_BYTES<D> + (((c & 7) ^ row_swizzle<D>(r)) << 4); }
// the address of chunk 2 x + b from that of chunk b of the same row (blocks begin at multiples of 128 bytes)
__device__ __forceinline__ uint32_t chunk_pair(uint32_t a, int x) { return (a ^ ((x & 3) << 5)) + (x >> 2) * (KB * 128); }
__device__ __forceinline__ float2 load2_as_f(const void* base, int type, int64_t i) {
  if (type == B200Q_F32) return make_float2(static_cast<const float*>(base)[i], static_cast<const float*>(base)[i + 1]);
  const uint16_t* p = static_cast<const uint16_t*>(base) + i;
  return unpack2(p[0] | (uint32_t)p[1] << 16, type == B200Q_BF16);
}

template <int D, int N, bool BF, bool BOXES>
__device__ __forceinline__ void attn_rows(const AttnParams& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v) {
  constexpr int R = 16, CH = D / 8, ST = R_STAGES<D>, BLOCK = R_BLOCK<D>, KK = D / 16, PP = D >= 64 ? D / 64 : 1;
  extern __shared__ unsigned char raw[];
  __shared__ float s_m[RW][R], s_l[RW][R], s_scale[R];
  __shared__ uint64_t s_full[RW][ST];
  __shared__ int s_flag, s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
  const uint32_t s_ring = (s_addr(raw) + 1023) & ~1023u, s_q = s_ring + R_RING<D>, base = s_ring + warp * (ST * 2 * BLOCK);
  float* const s_o = reinterpret_cast<float*>(raw + (s_ring - s_addr(raw)));       // [warp][R][D]
  if constexpr (BOXES) {
    if (tid == 0) s_abort = 0;
    if (lane < ST) a_bar_init(&s_full[warp][lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async();
  }
  // Behind the tiles kernel of the same call (late): both read what was there before that one began and write rows of their own, so that this one waits for it only at its end.
  // (The fence: what is read now must not come from a first-level cache that has seen an earlier call's values.)
  if (p.late) __threadfence();
  else pdl_wait();
  pdl_launch_dependents();
  const int ps = p.t.page_size;
  const bool whole = BOXES || ps % KB == 0;              // a block lies in one page

  // ---- this CTA's share ----
  auto units_of = [&](const SeqPlace& q) { return (uint32_t)((unsigned)(q.n * p.group + R - 1) / R * p.n_kv); };
  auto rounds_of = [&](const SeqPlace& q) { return (uint32_t)max(1, (q.cap + ROUND - 1) / ROUND); };      // (without keys: somebody writes the zeros)
  struct Work { uint32_t units, rounds; };
  bool back = false;                                     // row_off goes back: sequences may overlap
  uint64_t rounds = 0;                                   // of this lane's sequences
  auto sums_of = [&](int s) {                            // of this lane's sequence and those of the lanes before it
    Work v{0, 0};
    if (s < p.t.n_seqs) {
      back |= p.t.row_off[s + 1] < p.t.row_off[s];
      const SeqPlace q = place_of_seq(p, s);
      if (blockIdx.x == 0 && warp == 0) check_place(p, s, q);
      v.units = units_of(q);
      v.rounds = v.units * rounds_of(q);
      rounds += (uint64_t)v.units * rounds_of(q);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, v.units, o), r = __shfl_up_sync(0xffffffffu, v.rounds, o);
      if (lane >= o) { v.units += u; v.rounds += r; }
    }
    return v;
  };
  Work sums{}, all{};
  for (int s0 = 0; s0 < p.t.n_seqs; s0 += 32) {
    sums = sums_of(s0 + lane);
    all.units += __shfl_sync(0xffffffffu, sums.units, 31);
    all.rounds += __shfl_sync(0xffffffffu, sums.rounds, 31);
  }
  // Sequences that overlap (check_place reports them) are work past the host's bound, which fits into 31 bits, and their sums may wrap around to units that no CTA ends, whose counters would wait for it in
  // the next call.
  if (__any_sync(0xffffffffu, back)) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rounds += __shfl_xor_sync(0xffffffffu, rounds, o);
    if (rounds > p.most_rounds) return;
  }
  // A unit costs its rounds and, where shares are long, what it takes to begin and end one.  A share that would begin or end in that part does so where the unit begins.
  const uint32_t ctas = min(gridDim.x, max(min(all.rounds, (uint32_t)N_SM), all.rounds / R_LEAST)), c = blockIdx.x;
  if (c >= ctas) return;
  const uint32_t extra = all.rounds / ctas >= R_LONG ? R_EXTRA : 0, total = all.rounds + extra * all.units;
  const uint32_t share = total / ctas, more = total - share * ctas, x_end = (c + 1) * share + min(c + 1, more);      // one more for the first `more` CTAs
  uint32_t x = c * share + min(c, more);
  auto cta_of = [&](uint32_t y) { return y < more * (share + 1) ? y / (share + 1) : more + (y - more * (share + 1)) / share; };
  int seq = 0;
  uint32_t seq_begin = 0;
  for (int s0 = 0; s0 < p.t.n_seqs; s0 += 32) {
    if (p.t.n_seqs > 32) sums = sums_of(s0 + lane);
    const uint32_t upto = sums.rounds + extra * sums.units;
    const unsigned here = __ballot_sync(0xffffffffu, x < seq_begin + upto);
    if (here) {
      const int l = __ffs(here) - 1;
      seq = s0 + l;
      if (l) seq_begin += __shfl_sync(0xffffffffu, upto, l - 1);
      break;
    }
    seq_begin += __shfl_sync(0xffffffffu, upto, 31);
  }
  SeqPlace sp = place_of_seq(p, seq);
  uint32_t n_issued = 0, n_used = 0;                     // this warp's blocks so far: stage and phase

#pragma unroll 1
  while (x < x_end) {
    // ---- the next unit of it ----
    uint32_t cost = rounds_of(sp) + extra;
    while (x >= seq_begin + units_of(sp) * cost) {
      seq_begin += units_of(sp) * cost;
      if (++seq >= p.t.n_seqs) return;                     // (sums of tables that contradict themselves)
      sp = place_of_seq(p, seq);
      cost = rounds_of(sp) + extra;
    }
    const uint32_t in_seq = (x - seq_begin) / cost, unit_begin = seq_begin + in_seq * cost, unit_end = unit_begin + cost, end = min(unit_end, x_end);
    const uint32_t from = x - unit_begin <= extra ? 0 : x - unit_begin - extra, to_round = end - unit_begin <= extra ? 0 : end - unit_begin - extra;
    if (to_round == 0) return;                             // the share ends in what it takes to begin: the next CTA begins there
    const int tile = p.by_kv.div(in_seq), kvh = in_seq - tile * p.n_kv;
    const TilePlace w = tile_of_seq<R>(p, seq, sp, tile);
    const int k_begin = from * ROUND, k_end = min((uint32_t)w.keys, to_round * ROUND), pairs = w.n * p.group;      // (rounds x 64 < 2^31 + 64)
    const int blocks = max(0, (k_end - k_begin + KB - 1) / KB), mine = (blocks - warp + RW - 1) / RW;      // this warp's: warp, warp + RW, ...
    auto block_key = [&](int it) { return k_begin + (warp + it * RW) * KB; };
    auto page_id = [&](int it) { return whole && it < mine ? p.t.pages[(int64_t)seq * p.t.table_stride + p.by_page.div(block_key(it))] : -1; };
    int ids = page_id(lane), ids_next = mine > 32 ? page_id(32 + lane) : 0;      // pages of this and the next 32 blocks

    // the queries, four rows a warp: all loads, then (behind the first blocks' copies) a power of two that keeps a row in fp16's range (N == 2) and their parts
    float2 f[4][PP];
    {
      int64_t at[4];
      bool live[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int pair = w.r0 + warp * 4 + i, token = p.by_group.div(pair);
        live[i] = pair < pairs && lane < D / 2;
        at[i] = (w.first_row + token) * p.q_stride + (kvh * p.group + pair - token * p.group) * D + lane * 2;
      }
      const int size = type_size(p.q_dtype);
      const bool paired = (((uintptr_t)p.q | (uintptr_t)(p.q_stride * size)) & (2 * size - 1)) == 0;
      if (p.q_dtype == B200Q_F32 && paired) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < PP; j++) f[i][j] = live[i] ? *reinterpret_cast<const float2*>(static_cast<const float*>(p.q) + at[i] + j * 64) : make_float2(0.f, 0.f);
      } else if (paired) {
        uint32_t v[4][PP];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < PP; j++) v[i][j] = live[i] ? *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.q) + at[i] + j * 64) : 0u;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < PP; j++) f[i][j] = unpack2(v[i][j], p.q_dtype == B200Q_BF16);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < PP; j++) f[i][j] = live[i] ? load2_as_f(p.q, p.q_dtype, at[i] + j * 64) : make_float2(0.f, 0.f);
      }
    }
    auto issue = [&](int it) {
      if (it < mine) {
        const int key0 = block_key(it);
        const uint32_t to = base + n_issued % ST * (2 * BLOCK);
        int page = 0;
        if (whole) {
          page = __shfl_sync(0xffffffffu, ids, it & 31);
          if ((it & 31) == 31) { ids = ids_next; ids_next = mine > it + 33 ? page_id(it + 33 + lane) : 0; }
          if ((unsigned)page >= (unsigned)p.t.n_pages) {
            if (lane == 0) atomicExch(&g_paged_attn_status, 2);
            page = BOXES ? p.t.n_pages : -1;               // (outside the map: the box is filled with zeros)
          }
        }
        if constexpr (BOXES) {
          const uint32_t bar = s_addr(&s_full[warp][n_issued % ST]);
          if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2 * BLOCK) : "memory");
          __syncwarp();
          if (lane < D / 32) {      // a lane a box: keys' sub-blocks, values' sub-blocks
            const int sub = lane % (D / 64);
            asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                         ::"r"(to + lane * (KB * 128)), "l"(lane < D / 64 ? &tm_k : &tm_v), "r"(bar), "r"(sub * 64), "r"(key0 - p.by_page.div(key0) * ps), "r"(kvh), "r"(page) : "memory");
          }
        } else {
          const uint16_t* kp = static_cast<const uint16_t*>(p.k) + kvh * p.head_stride;
          const uint16_t* vp = static_cast<const uint16_t*>(p.v) + kvh * p.head_stride;
          const int64_t at0 = page >= 0 ? page * p.page_stride + (int64_t)(key0 - p.by_page.div(key0) * ps) * p.row_stride : 0;
#pragma unroll
          for (int i = 0; i < (KB * CH + 31) / 32; i++) {
            const int ch = lane + i * 32, r = ch / CH, col = ch % CH;
            bool there = page >= 0 && key0 + r < k_end;
            int64_t at = at0 + (int64_t)r * p.row_stride;
            if (!whole) { at = there ? key_at(p, w.seq, key0 + r) : -1; there = at >= 0; }
            at = there ? at + col * 8 : 0;
            const uint32_t o = to + chunk_at<D>(r, col);
            copy16(o, kp + at, there ? 16 : 0);              // (nothing there: zeros)
            copy16(o + BLOCK, vp + at, there ? 16 : 0);
          }
        }
        n_issued++;
      }
      if constexpr (!BOXES) asm volatile("cp.async.commit_group;" ::: "memory");
    };

    uint32_t qa[N][KK][4];
    float qs[2];
    int last[2];                                           // the position a row may see up to
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    const int first_last = w.length + p.by_group.div(w.r0);      // what the tile's first row sees: blocks up to it are seen by all
#pragma unroll 1
    for (int it = 1 - ST; it < max(mine, 1); it++) {       // (one copy of the loop's code: what a short call waits for is instructions)
      if (it == 0) {
        // the first blocks are on their way: the queries' parts, in the order that ldmatrix puts into the instruction's A operand
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int r = warp * 4 + i;
          float up = 1.f, down = 1.f;
          if (N == 2) {
            float amax = 0.f;
#pragma unroll
            for (int j = 0; j < PP; j++) amax = fmaxf(amax, fmaxf(fabsf(f[i][j].x), fabsf(f[i][j].y)));
            amax = warp_max(amax);
            pow2_scale(amax, up, down);
            if (amax == 0.f) down = 1.f;
          }
          if (lane == 0) s_scale[r] = fmaxf(p.scale * down, 1.1754944e-38f);      // (scores of masked keys are -infinity times it)
#pragma unroll
          for (int j = 0; j < PP; j++) {
            uint32_t v[N];
            parts_of<N, BF>(f[i][j].x * up, f[i][j].y * up, v);
            if (lane < D / 2)
#pragma unroll
              for (int q = 0; q < N; q++)
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(s_q + q * (R * D * 2) + chunk_at<D>(r, lane / 4 + j * 8) + (lane & 3) * 4), "r"(v[q]) : "memory");
          }
        }
        __syncthreads();
        const uint32_t a = s_q + chunk_at<D>((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
#pragma unroll
        for (int q = 0; q < N; q++)
#pragma unroll
          for (int kk = 0; kk < KK; kk++) ldsm4(qa[q][kk], chunk_pair(a + q * (R * D * 2), kk));
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int pair = w.r0 + g + e * 8;
          last[e] = pair < pairs ? w.length + p.by_group.div(pair) : -1;
          qs[e] = s_scale[g + e * 8];
        }
        if (mine <= 0) break;
      }
      if (it >= 0) {
        if constexpr (BOXES) { if (!bar_ready(&s_full[warp][n_used % ST], n_used / ST & 1)) a_wait_on(s_addr(&s_full[warp][n_used % ST]), n_used / ST & 1, s_addr(&s_abort)); }
        else asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
        __syncwarp();
      }
      issue(it + ST - 1);
      if (it < 0) continue;
      const uint32_t ks = base + n_used % ST * (2 * BLOCK), vs = ks + BLOCK;
      n_used++;
      const int key0 = block_key(it);
      float s[2][4];
      {
        const uint32_t a = ks + chunk_at<D>((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1);
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
          uint32_t b[4];
          ldsm4(b, chunk_pair(a, kk));
#pragma unroll
          for (int i = N - 1; i >= 0; i--) {
            if (kk == 0 && i == N - 1) { mma_row0<BF>(s[0], qa[i][kk], b[0], b[1]); mma_row0<BF>(s[1], qa[i][kk], b[2], b[3]); }
            else { mma_row<BF>(s[0], qa[i][kk], b[0], b[1]); mma_row<BF>(s[1], qa[i][kk], b[2], b[3]); }
          }
        }
      }
      const bool masked = key0 + KB - 1 > first_last || key0 + KB > k_end;
      if (masked) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int key = key0 + j * 8 + tq * 2 + (e & 1);
            if (key > last[e >> 1] || key >= k_end) s[j][e] = -INFINITY;
          }
      }
      float cf[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float mx = fmaxf(fmaxf(s[0][e * 2], s[0][e * 2 + 1]), fmaxf(s[1][e * 2], s[1][e * 2 + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx = fmaxf(mx * qs[e], m[e]);
        cf[e] = mx == -INFINITY ? 1.f : pow2(m[e] - mx);
        m[e] = mx;
        const float sub = mx == -INFINITY ? 0.f : 14.f - mx;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int i = 0; i < 2; i++) s[j][e * 2 + i] = pow2(fmaf(s[j][e * 2 + i], qs[e], sub));
        l[e] = fmaf(l[e], cf[e], (s[0][e * 2] + s[0][e * 2 + 1]) + (s[1][e * 2] + s[1][e * 2 + 1]));
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
        if (BOXES && key0 + KB > k_end) {      // what the page holds behind the last key
          for (int i = lane; i < KB * CH; i += 32)
            if (key0 + i / CH >= k_end) st_s4(vs + chunk_at<D>(i / CH, i % CH), make_uint4(0, 0, 0, 0));
          __syncwarp();
        }
        for (int i = lane; i < KB * CH; i += 32) {
          uint32_t y[4];
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(y[0]), "=r"(y[1]), "=r"(y[2]), "=r"(y[3]) : "r"(vs + i * 16) : "memory");
#pragma unroll
          for (int j = 0; j < 4; j++) odd |= finite_only<BF>(y[j]) != y[j];
        }
        odd = __any_sync(0xffffffffu, odd);
      }
      const uint32_t va = vs + chunk_at<D>((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
#pragma unroll
      for (int n = 0; n < D / 16; n++) {
        uint32_t b[4];
        ldsm4_t(b, chunk_pair(va, n));
        if (odd) {
#pragma unroll
          for (int j = 0; j < 4; j++) b[j] = finite_only<BF>(b[j]);
        }
        float t[2][4];
        mma_row0<BF>(t[0], pa[N - 1], b[0], b[1]);
        mma_row0<BF>(t[1], pa[N - 1], b[2], b[3]);
#pragma unroll
        for (int i = N - 2; i >= 0; i--) { mma_row<BF>(t[0], pa[i], b[0], b[1]); mma_row<BF>(t[1], pa[i], b[2], b[3]); }
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[2 * n + y][e] = fmaf(o[2 * n + y][e], cf[e >> 1], t[y][e]);
      }
      if (odd) {             // what was left out, for the rows that see it (the others keep their bits)
#pragma unroll 1
        for (int j = 0; j < KB; j++) {
          float e2[2];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int from = (lane & ~3) | (j & 7) / 2;
            float y[4];
#pragma unroll
            for (int q = 0; q < 4; q++) y[q] = __shfl_sync(0xffffffffu, s[q >> 1][e * 2 + (q & 1)], from);
            e2[e] = j < 8 ? (j & 1 ? y[1] : y[0]) : j & 1 ? y[3] : y[2];
          }
          const bool sees[2] = {key0 + j <= last[0], key0 + j <= last[1]};
#pragma unroll
          for (int n = 0; n < D / 8; n++) {
            uint32_t y;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(y) : "r"(vs + chunk_at<D>(j, n) + tq * 4) : "memory");
            const uint32_t left = y ^ finite_only<BF>(y);      // the values that are not finite, zeros elsewhere
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
    if constexpr (!BOXES) asm volatile("cp.async.wait_group 0;" ::: "memory");

    // the warps' sums, in the order of the warps
#pragma unroll
    for (int e = 0; e < 2; e++) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if (tq == 0) { s_m[warp][g + e * 8] = m[e]; s_l[warp][g + e * 8] = l[e]; }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int r = g + e * 8;
      const float cw = l[e] == 0.f ? 0.f : pow2(m[e] - fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r])));
#pragma unroll
      for (int n = 0; n < D / 8; n++) *reinterpret_cast<float2*>(s_o + (warp * R + r) * D + n * 8 + tq * 2) = make_float2(l[e] == 0.f ? 0.f : o[n][e * 2] * cw, l[e] == 0.f ? 0.f : o[n][e * 2 + 1] * cw);
    }
    __syncthreads();
    const int c_first = cta_of(unit_begin + extra), n_parts = cta_of(unit_end - 1) - c_first + 1;
    auto place = [&](int cta, bool first) { return p.parts + (cta * 2 + first) * PART<R, D>; };
    float* const part = place(c, from == 0);
#pragma unroll 1
    for (int i = tid; i < R * D / 4; i += R_THREADS) {
      const int r = i / (D / 4), d = (i - r * (D / 4)) * 4, pair = w.r0 + r;
      if (pair >= pairs) break;
      float ml = -INFINITY, sum = 0.f, v[4] = {};
#pragma unroll
      for (int q = 0; q < RW; q++) ml = fmaxf(ml, s_m[q][r]);
#pragma unroll
      for (int q = 0; q < RW; q++) {
        const float lx = s_l[q][r];
        sum += lx == 0.f ? 0.f : lx * pow2(s_m[q][r] - ml);
        const float4 y = *reinterpret_cast<const float4*>(s_o + (q * R + r) * D + d);
        v[0] += y.x; v[1] += y.y; v[2] += y.z; v[3] += y.w;
      }
      if (n_parts == 1) {
        const int token = p.by_group.div(pair);
        const int64_t at = (w.first_row + token) * p.out_stride + (kvh * p.group + pair - token * p.group) * D + d;
#pragma unroll
        for (int j = 0; j < 4; j++) store_as(p.out, p.out_dtype, at + j, sum == 0.f ? 0.f : v[j] / sum);
      } else {
        if (d == 0) { __stcg(part + r, ml); __stcg(part + R + r, sum); }
        __stcg(reinterpret_cast<float4*>(part + 2 * R + r * D + d), make_float4(v[0], v[1], v[2], v[3]));
      }
    }
    if (n_parts > 1) join_parts<R, D, R_THREADS>(p, w, p.counters + c_first, n_parts, kvh, &s_flag, s_o, [&](int q) { return place(c_first + q, q == 0); });
    x = end;
    if constexpr (BOXES) fence_async();      // (what comes next into the ring comes through the other proxy)
    __syncthreads();
  }
}

template <int D, int N, bool BF, bool BOXES>
__global__ void __launch_bounds__(R_THREADS, 2) attn_rows_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  attn_rows<D, N, BF, BOXES>(p, tm_k, tm_v);
  if (p.late) pdl_wait();
}

// The map of a pool: [page][KV head][slot][value], boxes of 64 values x box_rows slots in the 128-byte-swizzle layout.
int make_page_map(CUtensorMap* tm, const b200q_paged_cache* c, const void* pool, int box_rows) {
  typedef CUresult (*encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<encode_fn> known{nullptr};
  encode_fn fn = known.load(std::memory_order_acquire);
  if (!fn) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    B200Q_CHECK_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q));
    if (!f || q != cudaDriverEntryPointSuccess) return B200Q_ERR_UNSUPPORTED;
    known.store(fn = (encode_fn)f, std::memory_order_release);
  }
  const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size, (cuuint64_t)c->n_kv_heads, (cuuint64_t)c->n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)c->row_stride * 2, (cuuint64_t)c->head_stride * 2, (cuuint64_t)c->page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, ones[4] = {1, 1, 1, 1};
  const CUresult r = fn(tm, c->dtype == B200Q_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(pool), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200Q_OK : B200Q_ERR_UNSUPPORTED;
}


}  // namespace
