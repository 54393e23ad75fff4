// Attention of a batch's new tokens over a paged KV cache (tinygrad/llm/model.py:187-195 with a cache of pages and sequences of different lengths).
//   row (token i of n, query head h), position p = length - n + i:  out = sum_{j <= p} e^(s_j - m) v_j / sum_{j <= p} e^(s_j - m),  s_j = scale q . k_j,  m = max s_j,
// in one pass over the keys with the running maximum and sums of the softmax (32-bit); KV head h / G serves the G query heads of its group.
//
// Work is dealt as (tile of rows, KV head, part of the keys).  A tile is R consecutive (token, head of the group) pairs of one sequence, token-major, so the group's heads share every key
// that is loaded.  Three kernels share the work: sequences of few rows (paged_attn_rows.cuh), of many (paged_attn_tiles.cuh), and what neither takes (fp32 pages; below).  The keys are split over
// CTAs where the tiles alone do not fill the GPU: parts leave (m, sum, weighted sum) in the workspace, and the one that is done last (a kernel behind it, for the tiles of many rows)
// adds them in the order of the keys, so that results do not depend on timing, and puts the counter back.
#include "paged.cuh"
#include <algorithm>

namespace {

__device__ int g_paged_attn_status = 0;

constexpr int N_SM = 148;      // of a B200
constexpr float LOG2E = 1.4426950408889634f;

struct AttnParams {
  const void *q, *k, *v;
  void* out;
  int q_dtype, out_dtype;
  int64_t q_stride, out_stride, page_stride, head_stride, row_stride;
  int n_kv, group;
  float scale;               // times log2 e
  Divisor by_group, by_kv, by_page;
  int tiles_per_seq;         // 0: tiles are counted sequence by sequence
  int above, up_to;          // sequences with above < new tokens <= up_to (those with others are another kernel's)
  int n_split, split_len, late;      // late: behind the tiles kernel of the same call
  uint32_t most_rounds;      // of the rows kernel, by the host's bounds
  int* counters;
  float* parts;
  PagedTables t;
};

struct TilePlace { int seq, first_row, n, r0, length, keys; };       // r0: the tile's first (token, head) pair; keys: those its last row sees, at most

// A sequence's rows, those of them that this kernel has, its positions that may be attended, the position of its first new token
struct SeqPlace { int first_row, n, cap, start; };
__device__ __forceinline__ SeqPlace place_of_seq(const AttnParams& p, int s) {
  const PagedTables& t = p.t;
  const int b0 = t.row_off[s], e0 = t.row_off[s + 1], length = t.length[s];
  const int b = min(max(b0, 0), t.n_rows), e = min(max(e0, b), t.n_rows), n = min(e - b, t.max_new);
  const int64_t room = (int64_t)t.table_stride * t.page_size;
  return SeqPlace{b, n > p.above && n <= p.up_to ? n : 0, (int)min((int64_t)min(max(length, 0), t.max_len), room), length - (e0 - b)};      // (by all of its rows, those past the arrays among them)
}
__device__ __forceinline__ bool rows_outside(const PagedTables& t, int s) {      // rows that go back, or that the arrays do not have
  const int b = t.row_off[s], e = t.row_off[s + 1];
  return e < b || b < 0 || e > t.n_rows;
}
__device__ __forceinline__ void check_place(const AttnParams& p, int s, const SeqPlace& q) {      // what the tables promise and the bounds do not hold
  if (rows_outside(p.t, s) || (q.n > 0 && (p.t.row_off[s + 1] - q.first_row > q.n || p.t.length[s] > q.cap))) atomicExch(&g_paged_attn_status, 2);
}
template <int R>
__device__ __forceinline__ TilePlace tile_of_seq(const AttnParams& p, int s, const SeqPlace& q, int tile) {
  TilePlace w{s, q.first_row, q.n, tile * R, q.start, 0};
  const int last = min(p.by_group.div(w.r0 + R - 1), q.n - 1);
  w.keys = max(0, min(q.cap, q.start + last + 1));
  return w;
}

// R pairs to a tile; by a whole warp.  n == 0: nothing to do.
template <int R>
__device__ __forceinline__ TilePlace place_of_tile(const AttnParams& p, int tile) {
  const PagedTables& t = p.t;
  const int lane = threadIdx.x & 31;
  int s = 0;
  if (p.tiles_per_seq) {
    s = tile / p.tiles_per_seq;
    tile -= s * p.tiles_per_seq;
  } else {
    bool found = false;
    for (int s0 = 0; s0 < t.n_seqs && !found; s0 += 32) {
      if (s0 + lane < t.n_seqs && rows_outside(t, s0 + lane)) atomicExch(&g_paged_attn_status, 2);
      const int mine = s0 + lane < t.n_seqs ? (place_of_seq(p, s0 + lane).n * p.group + R - 1) / R : 0;
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += u; }
      const unsigned here = __ballot_sync(0xffffffffu, tile < sum);
      if (here) {
        const int l = __ffs(here) - 1;
        s = s0 + l;
        tile -= __shfl_sync(0xffffffffu, sum - mine, l);
        found = true;
      } else tile -= __shfl_sync(0xffffffffu, sum, 31);
    }
    if (!found) return TilePlace{};
  }
  const SeqPlace q = place_of_seq(p, s);
  if (lane == 0 && tile == 0) check_place(p, s, q);
  if (tile * R >= q.n * p.group) return TilePlace{};
  return tile_of_seq<R>(p, s, q, tile);
}

// the offset of a key in the pages, or -1
__device__ __forceinline__ int64_t key_at(const AttnParams& p, int seq, int key) {
  const int index = key / p.t.page_size, page = p.t.pages[(int64_t)seq * p.t.table_stride + index];
  if (page < 0 || page >= p.t.n_pages) { atomicExch(&g_paged_attn_status, 2); return -1; }
  return page * p.page_stride + (int64_t)(key - index * p.t.page_size) * p.row_stride;
}

// ---- parts of the keys ----  (a sum of a length and a part's may pass 31 bits)
__device__ __forceinline__ int parts_of_keys(const AttnParams& p, int keys) { return keys > 0 ? (keys - 1) / p.split_len + 1 : 1; }
template <int R, int D> constexpr int PART = R * (D + 2);           // m [R], sum [R], weighted sum [R][D]

// The tile's last part to be done adds all of them; by the whole CTA (THREADS).  m in log2.  One thread's count releases what all have stored before the barrier.  Then the first AHEAD parts of every
// thread's values are asked for, every part's share of each row is computed meanwhile (a warp a row, a lane a part), and the values are added.  factors: shared, R x n_parts.
// part_at(s): where part s is.  (One value after the other, 513 positions took 16 us more; with a fence in every thread and the values behind the shares 2 us more.)
template <int R, int D, int THREADS, typename At>
__device__ __forceinline__ void join_parts(const AttnParams& p, const TilePlace& w, int* counter, int n_parts, int kvh, int* s_flag, float* factors, At part_at) {
  constexpr int AHEAD = 4;
  __syncthreads();
  if (threadIdx.x == 0) {
    int old;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
    *s_flag = old == n_parts - 1;
    if (old == n_parts - 1) *counter = 0;
  }
  __syncthreads();
  if (!*s_flag) return;
  const int lane = threadIdx.x & 31, live = min(R, w.n * p.group - w.r0);
  float4 ahead[AHEAD];
  auto value = [&](int i, int s) { return __ldcg(reinterpret_cast<const float4*>(part_at(s) + 2 * R + i * 4)); };
  if ((int)threadIdx.x < live * (D / 4)) {
#pragma unroll
    for (int s = 0; s < AHEAD; s++) ahead[s] = value(threadIdx.x, min(s, n_parts - 1));
  }
  for (int r = threadIdx.x >> 5; r < live; r += THREADS / 32) {
    float m = -INFINITY, sum = 0.f, m0 = -INFINITY, l0 = 0.f;
    if (lane < n_parts) { m0 = __ldcg(part_at(lane) + r); l0 = __ldcg(part_at(lane) + R + r); }
    m = m0;
    for (int s = lane + 32; s < n_parts; s += 32) m = fmaxf(m, __ldcg(part_at(s) + r));
    m = warp_max(m);
    const float f0 = l0 == 0.f ? 0.f : exp2f(m0 - m);      // (a part without keys has sum 0)
    sum = f0 * l0;
    for (int s = lane + 32; s < n_parts; s += 32) {
      const float ls = __ldcg(part_at(s) + R + r), f = ls == 0.f ? 0.f : exp2f(__ldcg(part_at(s) + r) - m);
      factors[s * R + r] = f;
      sum = fmaf(f, ls, sum);
    }
    sum = warp_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (lane < n_parts) factors[lane * R + r] = f0 * inv;
    for (int s = lane + 32; s < n_parts; s += 32) factors[s * R + r] *= inv;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < live * (D / 4); i += THREADS) {
    const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
    float o[4] = {};
    auto add = [&](float4 v, int s) {
      const float f = factors[s * R + r];
      o[0] = fmaf(f, v.x, o[0]); o[1] = fmaf(f, v.y, o[1]); o[2] = fmaf(f, v.z, o[2]); o[3] = fmaf(f, v.w, o[3]);
    };
    int s0 = 0;
    if (i == (int)threadIdx.x) {
#pragma unroll
      for (int s = 0; s < AHEAD; s++)
        if (s < n_parts) add(ahead[s], s);
      s0 = AHEAD;
    }
#pragma unroll 8
    for (int s = s0; s < n_parts; s++) add(value(i, s), s);
    const int pair = w.r0 + r, token = p.by_group.div(pair);
    const int64_t at = (w.first_row + token) * p.out_stride + (int64_t)(kvh * p.group + pair - token * p.group) * D + d;
#pragma unroll
    for (int j = 0; j < 4; j++) store_as(p.out, p.out_dtype, at + j, o[j]);
  }
}

// ---- any types: multiply-adds in 32 bits.  A warp takes every fourth block of 32 keys, a key a lane for the scores, D / 32 values a lane for the weighted sum. ----
constexpr int S_R = 16, S_WARPS = 4, S_THREADS = S_WARPS * 32;
template <int D, typename KV>
__global__ void __launch_bounds__(S_THREADS) attn_simple_kernel(const AttnParams p) {
  constexpr int R = S_R, NV = D >= 32 ? D / 32 : 1, LIVE = D >= 32 ? 32 : D;
  __shared__ float s_q[R][D], s_p[S_WARPS][R][32], s_o[R][D], s_m[S_WARPS][R], s_l[S_WARPS][R];
  __shared__ int s_flag;
  extern __shared__ float s_f[];      // shares of the parts
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y, split = blockIdx.z;
  const TilePlace w = place_of_tile<R>(p, blockIdx.x);
  if (w.n == 0) return;
  const int n_parts = parts_of_keys(p, w.keys), k_begin = split * p.split_len, k_end = k_begin + min(w.keys - k_begin, p.split_len);
  if (split >= n_parts) return;
  const int64_t pairs = (int64_t)w.n * p.group;
  for (int i = tid; i < R * D; i += S_THREADS) {
    const int r = i / D, d = i - r * D, pair = w.r0 + r, token = pair / p.group;
    s_q[r][d] = pair < pairs ? load_as_f(p.q, p.q_dtype, (w.first_row + token) * p.q_stride + (int64_t)(kvh * p.group + pair - token * p.group) * D + d) * p.scale : 0.f;
    s_o[r][d] = 0.f;
  }
  __syncthreads();
  float o[R][NV], m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    m[r] = -INFINITY; l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++) o[r][j] = 0.f;
  }
  const KV* kp = static_cast<const KV*>(p.k) + kvh * p.head_stride;
  const KV* vp = static_cast<const KV*>(p.v) + kvh * p.head_stride;
  for (int k0 = k_begin + warp * 32; k0 < k_end; k0 += S_WARPS * 32) {
    const int key = k0 + lane;
    const int64_t at = key < k_end ? key_at(p, w.seq, key) : -1;
    float s[R];
#pragma unroll
    for (int r = 0; r < R; r++) s[r] = 0.f;
    for (int d = 0; d < D; d += 4) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (at >= 0) {
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = to_f(kp[at + d + j]);
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float4 q = *reinterpret_cast<const float4*>(&s_q[r][d]);
        s[r] = fmaf(q.x, f[0], fmaf(q.y, f[1], fmaf(q.z, f[2], fmaf(q.w, f[3], s[r]))));
      }
    }
    int first = w.length + w.r0 / p.group, h = w.r0 % p.group;        // the position and head of row r
    const bool all = k0 + 31 < k_end && k0 + 31 <= first;             // every row sees every key of the block
    __syncwarp();
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (key >= k_end || key > first) s[r] = -INFINITY;
      if (++h == p.group) { h = 0; first++; }
      const float mn = fmaxf(m[r], warp_max(s[r])), c = mn == -INFINITY ? 1.f : exp2f(m[r] - mn);
      const float e = mn == -INFINITY && s[r] == -INFINITY ? 0.f : exp2f(s[r] - mn);
      m[r] = mn;
      l[r] = l[r] * c + warp_sum(e);
#pragma unroll
      for (int j = 0; j < NV; j++) o[r][j] *= c;
      s_p[warp][r][lane] = s[r] == -INFINITY ? 0.f : e;
    }
    __syncwarp();
    const int n = min(32, k_end - k0);
    for (int j = 0; j < n; j++) {
      const int64_t vat = __shfl_sync(0xffffffffu, at, j);
      float f[NV];
#pragma unroll
      for (int i = 0; i < NV; i++) f[i] = vat >= 0 && lane < LIVE ? to_f(vp[vat + lane + i * 32]) : 0.f;
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float e = s_p[warp][r][j];
#pragma unroll
        for (int i = 0; i < NV; i++) o[r][i] = all || e != 0.f ? fmaf(e, f[i], o[r][i]) : o[r][i];      // (a masked value may be anything)
      }
    }
  }
  // the warps' sums, in the order of the warps
  if (lane == 0)
#pragma unroll
    for (int r = 0; r < R; r++) { s_m[warp][r] = m[r]; s_l[warp][r] = l[r]; }
  __syncthreads();
  float mt[R];
#pragma unroll
  for (int r = 0; r < R; r++) mt[r] = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
  for (int x = 0; x < S_WARPS; x++) {
    if (x == warp && lane < LIVE)
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float c = l[r] == 0.f ? 0.f : exp2f(m[r] - mt[r]);
#pragma unroll
        for (int i = 0; i < NV; i++) s_o[r][lane + i * 32] += o[r][i] * c;
      }
    __syncthreads();
  }
  const int unit = blockIdx.x * p.n_kv + kvh;
  float* mine = p.parts + ((int64_t)unit * p.n_split + split) * PART<R, D>;
  for (int i = tid; i < R * D; i += S_THREADS) {
    const int r = i / D, d = i - r * D, pair = w.r0 + r, token = pair / p.group;
    if (pair >= pairs) break;
    float ml = -INFINITY, sum = 0.f;
    for (int x = 0; x < S_WARPS; x++) ml = fmaxf(ml, s_m[x][r]);
    for (int x = 0; x < S_WARPS; x++) sum += s_l[x][r] == 0.f ? 0.f : s_l[x][r] * exp2f(s_m[x][r] - ml);
    if (n_parts == 1) {
      store_as(p.out, p.out_dtype, (w.first_row + token) * p.out_stride + (int64_t)(kvh * p.group + pair - token * p.group) * D + d, sum == 0.f ? 0.f : s_o[r][d] / sum);
    } else {
      if (d == 0) { __stcg(mine + r, ml); __stcg(mine + R + r, sum); }
      __stcg(mine + 2 * R + i, s_o[r][d]);
    }
  }
  const float* first = p.parts + (int64_t)unit * p.n_split * PART<R, D>;
  if (n_parts > 1) join_parts<R, D, S_THREADS>(p, w, p.counters + unit, n_parts, kvh, &s_flag, s_f, [&](int s) { return first + (int64_t)s * PART<R, D>; });
}

}  // namespace
#include "paged_attn_rows.cuh"
#include "paged_attn_tiles.cuh"
namespace {

// ---- how the work is dealt ----
// Positions that can be attended: the end of the last one's tile is an int.  Lengths past a bound of the host's are not attended and reported.
constexpr int MAX_KEYS = INT32_MAX - (T_KEYS - 1);
static_assert(T_KEYS % ROUND == 0, "rounds end inside");
b200q_paged_batch bounded(const b200q_paged_batch* b) {
  b200q_paged_batch c = *b;
  c.max_len = std::min(c.max_len, MAX_KEYS);
  return c;
}
constexpr int MAX_PARTS = 296;      // of the keys of a tile of 16 rows: their shares take 19 KB of shared memory (tiles of 256 rows have T_PARTS at most)
struct Plan { int64_t tiles; int tiles_per_seq, n_split, split_len, above, up_to, ctas; int64_t rounds; size_t bytes; };      // tiles x KV heads past 2^31 and rounds of -1: too large; bytes: of the parts in the workspace

// Tiles of `rows` pairs: those of all sequences at their largest, or (ragged batches, if that is less) the pairs' tiles and a broken one for each sequence.  Keys are split until
// there are about `want` CTAs, in parts of at least `least` keys.
Plan make_plan(const b200q_paged_cache* c, const b200q_paged_batch* b, int group, int above, int up_to, int rows, int want, int least, int unit, int most_parts) {
  const int n_kv = c->n_kv_heads, most_new = b->max_new < up_to ? b->max_new : up_to;
  const int64_t per = ((int64_t)most_new * group + rows - 1) / rows, even = per * b->n_seqs, ragged = (int64_t)b->n_rows * group / rows + b->n_seqs;
  Plan p{};
  p.above = above; p.up_to = up_to;
  p.tiles_per_seq = even <= ragged ? (int)per : 0;
  p.tiles = even <= ragged ? even : ragged;
  const int64_t len = b->max_len > 0 ? b->max_len : 1, most = (len + least - 1) / least;
  const int64_t parts = p.tiles > INT32_MAX / n_kv ? 0 : want / (p.tiles * n_kv);
  const int64_t n = std::min(std::max(std::min(parts, most), (int64_t)1), (int64_t)most_parts);
  p.split_len = (int)(((len + n - 1) / n + unit - 1) / unit * unit);
  p.n_split = (int)((len + p.split_len - 1) / p.split_len);      // at most want
  p.bytes = p.n_split == 1 ? 0 : ((size_t)p.tiles * n_kv * p.n_split * rows * (c->head_dim + 2) * 4 + 255) / 256 * 256;
  return p;
}

// The workspace begins with the counters of the tiles that are split, MAX_UNITS for each kernel of a call: a fixed place, whatever calls share the workspace.  Tiles x KV heads are split only
// where they are at most half of the CTAs that are wanted.
constexpr int MAX_UNITS = 2048, ROWS_CTAS = 2 * N_SM, MOST_CTAS = 4 * N_SM;
constexpr size_t COUNTERS_BYTES = 2 * MAX_UNITS * sizeof(int);
static_assert(MOST_CTAS / 2 <= MAX_UNITS && ROWS_CTAS <= MAX_UNITS, "counters");

// The rows kernel: as many CTAs as run at once, or as there is work for; parts of every CTA
Plan rows_plan(const b200q_paged_cache* c, const b200q_paged_batch* b, int group, int above, int up_to) {
  Plan p = make_plan(c, b, group, above, up_to, 16, 1, 1, ROUND, 1);
  p.rounds = p.tiles > INT32_MAX / c->n_kv_heads ? -1 : p.tiles * c->n_kv_heads * (std::max<int64_t>(1, ((int64_t)b->max_len + ROUND - 1) / ROUND) + R_EXTRA);
  p.ctas = (int)std::min<uint64_t>(p.rounds, ROWS_CTAS);
  p.bytes = (size_t)p.ctas * 2 * 16 * (c->head_dim + 2) * 4;
  return p;
}

// Batches whose sequences have at most ROWS_PAIRS (token, head) pairs each are the rows kernel's; in others it takes those of at most FEW_PAIRS.  It reads the keys again for every 16 pairs, mostly from L2; the tiles
// kernel's tiles are 256 pairs of which few may be rows, but another kernel for some of the sequences costs as well.  us, 8 sequences of up to 16 new tokens x 4 heads and 4000 positions: the rows kernel alone 43, both
// 72.  FEW_PAIRS 16 / 32 / 64 / 128: 8 of up to 32 tokens 52 / 69 / 74 / 62, 12 of up to 170 85 / 98 / 101 / 134, the same of fp32 rows 158 / 159 / 168 / 167, 12 of up to 700 and 3000 positions 52 / 52 / 52 / 68.
constexpr int ROWS_PAIRS = 64, FEW_PAIRS = 16;
// The kernels of a call and their shares of it.  many: there is work for the tiles kernel.
struct Deal { bool many; int n; Plan plan[2]; size_t bytes; };
Deal deal_of(const b200q_paged_cache* c, const b200q_paged_batch* b, int group, bool tiles_take) {
  Deal d{};
  const int few = FEW_PAIRS / group > 1 ? FEW_PAIRS / group : 1;
  d.many = tiles_take && (int64_t)b->max_new * group > ROWS_PAIRS && b->max_new > 1;
  if (d.many) {
    d.plan[0] = make_plan(c, b, group, few, INT32_MAX, T_R, N_SM, 512, T_KEYS, T_PARTS);
    d.n = 1;
    if (b->n_seqs > 1) {
      d.plan[1] = rows_plan(c, b, group, 0, few);
      d.n = 2;
    } else d.plan[0].above = 0;
  } else {
    d.plan[0] = c->dtype == B200Q_F32 ? make_plan(c, b, group, 0, INT32_MAX, S_R, MOST_CTAS, 256, 32, MAX_PARTS) : rows_plan(c, b, group, 0, INT32_MAX);
    d.n = 1;
  }
  const size_t parts = d.plan[0].bytes + d.plan[1].bytes;
  d.bytes = parts ? COUNTERS_BYTES + parts : 0;
  return d;
}
// TMA boxes of pages: 64 values x 16 positions (rows kernel), x a page's positions up to 128 (tiles kernel, whose tiles of 128 positions are whole boxes)
bool pages_have_boxes(const b200q_paged_cache* c) {
  return c->dtype != B200Q_F32 && c->head_dim >= 64 && c->page_size % KB == 0 && c->page_stride < (1LL << 38) && c->head_stride < (1LL << 38) && c->row_stride < (1LL << 38);
}
bool pages_for_tiles(const b200q_paged_cache* c) { return pages_have_boxes(c) && (c->page_size & (c->page_size - 1)) == 0; }
int box_rows_of(const b200q_paged_cache* c) { return c->page_size < T_KEYS ? c->page_size : T_KEYS; }

typedef void (*SimpleKernel)(const AttnParams);
typedef void (*RowsKernel)(const AttnParams, const CUtensorMap, const CUtensorMap);
constexpr int R_RING_OF[4] = {R_RING<16>, R_RING<32>, R_RING<64>, R_RING<128>};
typedef void (*TilesKernel)(const AttnParams, const CUtensorMap, const CUtensorMap, int);
SimpleKernel pick_simple(int dim) { return dim == 16 ? attn_simple_kernel<16, float> : dim == 32 ? attn_simple_kernel<32, float> : dim == 64 ? attn_simple_kernel<64, float> : attn_simple_kernel<128, float>; }
template <int D, bool BOXES>
RowsKernel pick_rows_of(int kv_dtype, int parts) {
  if (kv_dtype == B200Q_F16) return parts == 1 ? attn_rows_kernel<D, 1, false, BOXES> : attn_rows_kernel<D, 2, false, BOXES>;
  return parts == 1 ? attn_rows_kernel<D, 1, true, BOXES> : attn_rows_kernel<D, 3, true, BOXES>;
}
RowsKernel pick_rows(int dim, int kv_dtype, int parts, bool boxes) {
  if (dim == 128) return boxes ? pick_rows_of<128, true>(kv_dtype, parts) : pick_rows_of<128, false>(kv_dtype, parts);
  if (dim == 64) return boxes ? pick_rows_of<64, true>(kv_dtype, parts) : pick_rows_of<64, false>(kv_dtype, parts);
  return dim == 32 ? pick_rows_of<32, false>(kv_dtype, parts) : pick_rows_of<16, false>(kv_dtype, parts);
}
template <int D>
TilesKernel pick_tiles(int kv_dtype, int parts, int* smem) {
  *smem = parts == 1 ? T_SMEM<D, 1> : T_SMEM<D, 2>;
  if (kv_dtype == B200Q_F16) return parts == 1 ? attn_tiles_kernel<D, 1, false> : attn_tiles_kernel<D, 2, false>;
  return attn_tiles_kernel<D, 1, true>;
}
template <typename K>
int allow_smem(K kernel, int smem, PerDeviceFlag& flag) {
  const int dev = b200q_current_device();
  if (dev < 0) return B200Q_ERR_CUDA;
  if (flag.test(dev)) return B200Q_OK;
  B200Q_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  flag.set(dev);
  return B200Q_OK;
}

}  // namespace

int b200q_paged_attn_status_take(int* status) {
  int zero = 0;
  B200Q_CHECK_CUDA(cudaMemcpyFromSymbol(status, g_paged_attn_status, sizeof(int)));
  B200Q_CHECK_CUDA(cudaMemcpyToSymbol(g_paged_attn_status, &zero, sizeof(int)));
  return B200Q_OK;
}

extern "C" size_t b200q_paged_attention_workspace_bytes(const b200q_paged_cache* cache, const b200q_paged_batch* batch, int n_heads) {
  if (check_cache(cache) != B200Q_OK || check_batch(batch) != B200Q_OK || n_heads <= 0 || n_heads % cache->n_kv_heads || batch->n_seqs == 0 || batch->n_rows == 0) return 0;
  const int group = n_heads / cache->n_kv_heads;
  const b200q_paged_batch within = bounded(batch);
  const size_t a = deal_of(cache, &within, group, false).bytes, b = pages_for_tiles(cache) ? deal_of(cache, &within, group, true).bytes : 0;
  return a > b ? a : b;
}

extern "C" int b200q_paged_attention(const b200q_paged_cache* cache, const b200q_paged_batch* batch, const b200q_paged_attn_args* a, int flags, void* stream) {
  int rc = check_cache(cache);
  if (rc == B200Q_OK) rc = check_batch(batch);
  if (rc != B200Q_OK) return rc;
  if (!a || a->n_heads <= 0 || a->n_heads % cache->n_kv_heads || !type_known(a->q_dtype) || !type_known(a->out_dtype) || !(a->scale >= 0.f) || a->scale > 3.4e38f) return B200Q_ERR_BAD_ARG;
  const int dim = cache->head_dim, n_kv = cache->n_kv_heads, group = a->n_heads / n_kv;
  const int64_t row = (int64_t)a->n_heads * dim;
  if ((a->q_stride && a->q_stride < row) || (a->out_stride && a->out_stride < row) || row > INT32_MAX || (int64_t)batch->max_new * group > INT32_MAX - 1024) return B200Q_ERR_BAD_SHAPE;
  if (batch->n_seqs == 0 || batch->n_rows == 0) return B200Q_OK;
  if (!a->q || !a->out) return B200Q_ERR_BAD_ARG;
  if ((uintptr_t)a->q % type_size(a->q_dtype) || (uintptr_t)a->out % type_size(a->out_dtype) || (uintptr_t)a->workspace & 255) return B200Q_ERR_MISALIGNED;
  if (a->q == a->out && (a->q_dtype != a->out_dtype || (a->q_stride ? a->q_stride : row) != (a->out_stride ? a->out_stride : row))) return B200Q_ERR_BAD_ARG;      // rows would be overwritten before they are read
  const b200q_paged_batch within = bounded(batch);
  batch = &within;
  // one part of 16 bits where queries, keys and outputs have 16; two (bf16 keys: three, which the rows kernel has) where something is wider
  const int parts = a->q_dtype == cache->dtype && a->out_dtype != B200Q_F32 ? 1 : 2;
  alignas(64) CUtensorMap boxes[4];      // of the rows kernel and the tiles kernel, k and v each
  memset(boxes, 0, sizeof(boxes));
  bool have_boxes = pages_have_boxes(cache);
  Deal deal = deal_of(cache, batch, group, pages_for_tiles(cache) && (parts == 1 || cache->dtype == B200Q_F16));
  auto fits = [&](const Deal& d) {
    for (int i = 0; i < d.n; i++)
      if (d.plan[i].rounds < 0 || d.plan[i].rounds > INT32_MAX || d.plan[i].n_split > 65535 || n_kv > 65535 || d.plan[i].tiles > INT32_MAX / n_kv) return B200Q_ERR_TOO_LARGE;
    return a->workspace_bytes < d.bytes || (d.bytes && !a->workspace) ? B200Q_ERR_TOO_LARGE : B200Q_OK;
  };
  if ((rc = fits(deal)) != B200Q_OK) return rc;
  for (int i = 0; i < 4 && have_boxes; i++) {
    if (i < 2 ? deal.many && deal.n == 1 : !deal.many) continue;
    rc = make_page_map(boxes + i, cache, i & 1 ? cache->v : cache->k, i < 2 ? KB : box_rows_of(cache));
    if (rc == B200Q_ERR_UNSUPPORTED) { have_boxes = false; deal = deal_of(cache, batch, group, false); }      // strides that no map can have; b200q_paged_attention_workspace_bytes knows both deals
    else if (rc != B200Q_OK) return rc;
  }
  if ((rc = fits(deal)) != B200Q_OK) return rc;
  const cudaStream_t st = (cudaStream_t)stream;
  auto params = [&](int i, int late) {
    const Plan& plan = deal.plan[i];
    int* const counters = (int*)a->workspace + i * MAX_UNITS;
    float* const parts_at = (float*)((char*)a->workspace + COUNTERS_BYTES + (i ? deal.plan[0].bytes : 0));
    return AttnParams{a->q, cache->k, cache->v, a->out, a->q_dtype, a->out_dtype, a->q_stride ? a->q_stride : row, a->out_stride ? a->out_stride : row, cache->page_stride,
                       cache->head_stride, cache->row_stride, n_kv, group, (a->scale > 0.f ? a->scale : 1.f / sqrtf((float)dim)) * LOG2E, divisor_of(group), divisor_of(n_kv), divisor_of(cache->page_size), plan.tiles_per_seq, plan.above, plan.up_to,
                       plan.n_split, plan.split_len, late, (uint32_t)plan.rounds, counters, parts_at, tables_of(cache, batch)};
  };
  for (int i = 0; i < deal.n; i++) {
    // many rows first: once the last of their CTAs has a place, those for few rows begin where others leave room (12 sequences, 1 to 700 new of up to 3000 positions: 52 us, 60 the other way around)
    const Plan& plan = deal.plan[i];
    const AttnParams p = params(i, i > 0);
    const bool pdl = i > 0 || (flags & B200Q_FLAG_PDL);
    const int type = cache->dtype == B200Q_BF16;
    if (deal.many && i == 0) {
      int smem;
      const TilesKernel kernel = dim == 64 ? pick_tiles<64>(cache->dtype, parts, &smem) : pick_tiles<128>(cache->dtype, parts, &smem);
      static PerDeviceFlag allowed[2][2][2];
      if ((rc = allow_smem(kernel, smem, allowed[type][parts - 1][dim == 128])) != B200Q_OK) return rc;
      B200Q_CHECK_CUDA(launch_k(kernel, dim3((unsigned)plan.tiles * n_kv, plan.n_split), dim3(T_THREADS), (size_t)smem, st, pdl, p, boxes[2], boxes[3], box_rows_of(cache)));
      continue;
    }
    if (cache->dtype == B200Q_F32) {
      B200Q_CHECK_CUDA(launch_k(pick_simple(dim), dim3((unsigned)plan.tiles, n_kv, plan.n_split), dim3(S_THREADS), (size_t)(plan.n_split * S_R * 4), st, pdl, p));
      continue;
    }
    const int d = dim == 16 ? 0 : dim == 32 ? 1 : dim == 64 ? 2 : 3, smem = R_RING_OF[d] + (parts == 1 ? 1 : type ? 3 : 2) * 16 * dim * 2 + 1024;
    const RowsKernel kernel = pick_rows(dim, cache->dtype, parts, have_boxes);
    static PerDeviceFlag allowed[2][2][2][4];
    if ((rc = allow_smem(kernel, smem, allowed[have_boxes][type][parts - 1][d])) != B200Q_OK) return rc;
    B200Q_CHECK_CUDA(launch_k(kernel, dim3(plan.ctas), dim3(R_THREADS), (size_t)smem, st, pdl, p, boxes[0], boxes[1]));
  }
  if (deal.many && deal.plan[0].n_split > 1) {
    const Plan& plan = deal.plan[0];
    const AttnParams p = params(0, 0);
    B200Q_CHECK_CUDA(launch_k(dim == 64 ? join_tiles_kernel<64> : join_tiles_kernel<128>, dim3((unsigned)plan.tiles * n_kv, J_SLICES), dim3(J_THREADS), 0, st, true, p));
  }
  return B200Q_OK;
}
