"""The paged KV cache on the device against 64-bit numpy: appending (norms of heads, rotation, pages), attention of ragged batches, and both in a row."""
import numpy as np
import pytest
from gpu_util import need_gpu
from oracle import paged as ref

pytestmark = pytest.mark.gpu

EPS = {"float32": 2.0 ** -23, "float16": 2.0 ** -10, "bfloat16": 2.0 ** -7}
TINY = {"float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0}       # half a step of fp16's subnormals


def put(x, dtype):
  """values -> (device buffer, the values that it holds, float64)"""
  from tinygrad_b200.runtime import DeviceBuffer
  x = np.asarray(x)
  if dtype == "bfloat16":
    b = ref.bf16_bits(x.astype(np.float32))
    return DeviceBuffer.from_numpy(b), ref.bf16_values(b).astype(np.float64)
  with np.errstate(over="ignore"): a = x.astype(dtype)
  return DeviceBuffer.from_numpy(a), a.astype(np.float64)


def get(buf, shape, dtype):
  a = buf.numpy(shape, np.uint16 if dtype == "bfloat16" else np.dtype(dtype))
  return (ref.bf16_values(a) if dtype == "bfloat16" else a).astype(np.float64)


def table(rng, length, page_size, spare=3):
  """Pages of every sequence in random order -> (table, number of pages); entries behind a sequence's pages are no pages at all."""
  need = [-(-l // page_size) for l in length]
  order = rng.permutation(sum(need) + spare)
  t = np.full((len(length), max(need + [1])), -7, np.int32)
  at = 0
  for s, n in enumerate(need):
    t[s, :n] = order[at:at + n]
    at += n
  return t, sum(need) + spare


def i32(a):
  from tinygrad_b200.runtime import DeviceBuffer
  return DeviceBuffer.from_numpy(np.asarray(a, np.int32))


def cos_sin(rows, dim):
  a = np.arange(rows)[:, None] * (10000.0 ** (-np.arange(0, dim, 2) / dim))[None]
  return np.concatenate([np.cos(a), np.sin(a)], -1).astype(np.float32)


def layout(name, pages, heads, size, dim):
  """(strides, size of a pool in elements, where the pool begins in it)"""
  if name == "head-major": return (heads * size * dim, size * dim, dim), pages * heads * size * dim
  if name == "slot-major": return (heads * size * dim, dim, heads * dim), pages * heads * size * dim
  return (3 * heads * size * (dim + 8), size * (dim + 8), dim + 8), 3 * pages * heads * size * (dim + 8)      # rows with room between, every third page


def in_layout(flat, strides, pages, heads, size, dim):
  return np.lib.stride_tricks.as_strided(flat, (pages, heads, size, dim), tuple(s * flat.itemsize for s in (*strides, 1)))


def status():
  from tinygrad_b200 import runtime
  return runtime.device_status()


# ---- norms and rotation ----
# Tolerance: a value is one of a c - b s: both products' roundings, the sum's, and what a and b lost in the norm.  The 128 squares are added in a tree of 4 + 5 levels and a chain of at most 16
# (25 roundings of 2^-24, halved by the root), the mean, eps, root, quotient and two products add 6: below 24 x 2^-24 of |a| + |b|.  Then half a step of the output's type.
def close_rows(got, want, reach, dtype, what):
  tol = 24 * 2.0 ** -24 * reach + EPS[dtype] / 2 * (np.abs(want) + 24 * 2.0 ** -24 * reach) + TINY[dtype]
  bad = np.abs(got - want) > tol
  assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, worst {np.max(np.abs(got - want) / np.maximum(tol, 1e-300)):.2f} tolerances"


def reach_of(x, w, eps, rot):
  """|a| + |b| of every value's pair (itself where nothing is rotated)."""
  a = np.abs(ref.head_norm(x, w, eps))
  r = 0 if rot is None else rot.shape[-1] // 2
  both = a[..., :r] + a[..., r:2 * r]
  return np.concatenate([both, both, a[..., 2 * r:]], -1)


APPEND = [   # seqs' (new, length), heads, KV heads, dim, page size, rotated, types of x / q / pages, norms, layout
  ([(1, 1)], 4, 2, 64, 16, 64, "float32", "float32", "float16", "", "head-major"),
  ([(1, 513)], 32, 8, 128, 16, 128, "float32", "float32", "float16", "qk", "head-major"),
  ([(5, 9), (1, 40), (17, 17)], 6, 3, 128, 8, 64, "float32", "float16", "float32", "qk", "slot-major"),
  ([(3, 3), (33, 70), (0, 12), (2, 66)], 7, 1, 32, 5, 32, "float16", "float16", "float16", "k", "loose"),
  ([(129, 300)], 4, 4, 16, 1, 16, "bfloat16", "bfloat16", "bfloat16", "q", "head-major"),
  ([(1, 64)] * 37, 28, 4, 128, 64, 32, "bfloat16", "float32", "bfloat16", "qk", "loose"),
  ([(2, 1000), (40, 41)], 5, 5, 64, 100, 6, "float16", "float32", "float16", "qk", "slot-major"),      # pairs that are not on 16-byte boundaries
  ([(4, 4)], 3, 1, 128, 3, 0, "float32", "float32", "float16", "qk", "head-major"),                    # no rotation
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(case):
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer
  seqs, h, hk, d, ps, r, xt, qt, ct, norms, lay = APPEND[case]
  rng = np.random.default_rng(case)
  new, length = [n for n, _ in seqs], [l for _, l in seqs]
  off, n = np.concatenate([[0], np.cumsum(new)]), sum(new)
  t, n_pages = table(rng, length, ps)
  pad = 3                                     # rows of no sequence
  x, xv = put(rng.standard_normal((n + pad, h + 2 * hk, d)) * 2, xt)
  strides, size = layout(lay, n_pages, hk, ps, d)
  before = rng.standard_normal(size).astype(np.float32)
  (k, kv0), (v, vv0) = put(before, ct), put(before + 1, ct)
  q, q0 = put(np.full((n + pad, h, d), 7.0), qt)
  wq, wk = (None if c not in norms else rng.uniform(0.5, 1.5, d).astype(np.float16) for c in "qk")
  rope = cos_sin(max(length), r) if r else None
  dev = lambda a: None if a is None else DeviceBuffer.from_numpy(a)
  status()
  cache = paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v, strides=strides)
  batch = paged.PagedBatch(i32(off), i32(length), i32(t), n_rows=n + pad, max_new=max(new), max_len=max(length))
  paged.append(cache, batch, x, q, h, xt, q_dtype=qt, rope=dev(rope), q_norm=dev(wq), k_norm=dev(wk), norm_eps=1e-5)
  places = ref.rows_of(off, length)
  rot = rope[[p for _, p in places]] if r else None
  xs = xv[:n]
  got = get(q, (n + pad, h, d), qt)
  close_rows(got[:n], ref.rotate(ref.head_norm(xs[:, :h], wq, 1e-5), rot), reach_of(xs[:, :h], wq, 1e-5, rot), qt, "q")
  assert (got[n:] == 7).all(), "rows behind the last sequence are left as they were"
  kw, kr = ref.rotate(ref.head_norm(xs[:, h:h + hk], wk, 1e-5), rot), reach_of(xs[:, h:h + hk], wk, 1e-5, rot)
  kg, vg = get(k, (size,), ct), get(v, (size,), ct)
  for flat in (kg, vg): assert np.isfinite(flat).all()
  kp, vp = in_layout(kg, strides, n_pages, hk, ps, d), in_layout(vg, strides, n_pages, hk, ps, d)
  where = [(t[s, p // ps], p % ps) for s, p in places]
  pg, sl = (np.array(c, int) for c in zip(*where))
  close_rows(kp[pg, :, sl], kw, kr, ct, "k")
  vw = xs[:, h + hk:]
  assert (np.abs(vp[pg, :, sl] - vw) <= EPS[ct] / 2 * np.abs(vw) + TINY[ct]).all(), "v"
  kp[pg, :, sl], vp[pg, :, sl] = in_layout(kv0, strides, n_pages, hk, ps, d)[pg, :, sl], in_layout(vv0, strides, n_pages, hk, ps, d)[pg, :, sl]
  assert (kg == kv0).all() and (vg == vv0).all(), "everything else in the pools is as it was"
  assert status() == 0


def test_append_where_the_tables_are_wrong():
  """A page that does not exist, a position outside the table's row, before 0 or past the rotation's: no writes, status 2."""
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer
  rng = np.random.default_rng(5)
  h, hk, d, ps, n_pages = 2, 1, 32, 4, 6
  x, xv = put(rng.standard_normal((4, h + 2 * hk, d)), "float32")
  for length, t, zero in (([9, 3], [[0, 1, 6], [-1, 2, 3]], []), ([9, 3], [[0, 1], [-5, 3]], []), ([1, 9], [[4], [6]], [0]), ([30, 31], [[0, 1], [2, 3]], [0, 1, 2, 3])):
    status()
    cache = paged.PagedCache(n_pages, ps, hk, d, "float32")
    q = DeviceBuffer.empty((4, h, d), np.float32, zero=True)
    batch = paged.PagedBatch(i32([0, 2, 4]), i32(length), i32(t), n_rows=4, max_new=2, max_len=31)
    paged.append(cache, batch, x, q, h, rope=DeviceBuffer.from_numpy(cos_sin(12, d)))
    got = get(q, (4, h, d), "float32")
    assert [i for i in range(4) if (got[i] == 0).all()] == zero, (length, t)
    want = np.zeros((n_pages, ps))
    for s, p in ref.rows_of([0, 2, 4], length):
      if 0 <= p < 12 and p // ps < len(t[s]) and 0 <= t[s][p // ps] < n_pages: want[t[s][p // ps], p % ps] = 1
    for buf in (cache.k, cache.v): assert ((get(buf, (n_pages, ps, d), "float32") != 0).any(-1) == want).all(), (length, t)
    assert status() == 2


def test_append_in_place_and_strided():
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(2)
  h, hk, d, ps, n, stride = 3, 1, 64, 16, 21, 5 * 64 + 24
  x, xv = put(rng.standard_normal((n, stride)), "float16")
  cache = paged.PagedCache(4, ps, hk, d)
  batch = paged.PagedBatch(i32([0, n]), i32([n]), i32([[2, 0]]), n_rows=n, max_new=n, max_len=n)
  from tinygrad_b200.runtime import DeviceBuffer
  rope = cos_sin(n, d)
  paged.append(cache, batch, x, x, h, "float16", rope=DeviceBuffer.from_numpy(rope), x_stride=stride, q_stride=stride)
  got = get(x, (n, stride), "float16")
  xs = xv[:, :5 * d].reshape(n, 5, d)
  close_rows(got[:, :h * d].reshape(n, h, d), ref.rotate(xs[:, :h], rope), reach_of(xs[:, :h], None, 0, rope), "float16", "q")
  assert (got[:, h * d:] == xv[:, h * d:]).all()
  k = get(cache.k, (4, ps, d), "float16")
  close_rows(np.concatenate([k[2], k[0]])[:n, None], ref.rotate(xs[:, h:h + 1], rope), reach_of(xs[:, h:h + 1], None, 0, rope), "float16", "k")


@pytest.mark.parametrize("rows,h,hk,d,r,xt,ot,in_place", [(1, 32, 8, 128, 128, "float32", "float32", False), (300, 28, 4, 128, 0, "float16", "float16", True), (77, 5, 0, 64, 10, "bfloat16", "float32", False),
                                                         (9, 0, 3, 32, 32, "float32", "bfloat16", False), (2, 3, 3, 16, 8, "float16", "float16", True)])
def test_head_norm_rope(rows, h, hk, d, r, xt, ot, in_place):
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer
  rng = np.random.default_rng(rows)
  x, xv = put(rng.standard_normal((rows, h + 2 * hk + 1, d)) * 3, xt)
  stride = (h + 2 * hk + 1) * d
  out, ov = (x, xv) if in_place else put(np.full((rows, h + hk, d), 5.0), ot)
  wq, wk = (rng.uniform(0.5, 1.5, d).astype(np.float16) for _ in "qk")
  rope, pos = (cos_sin(50, r), rng.integers(0, 50, rows).astype(np.int32)) if r else (None, None)
  paged.head_norm_rope(x, out, rows, h, hk, d, xt, out_dtype=ot, q_norm=DeviceBuffer.from_numpy(wq), k_norm=DeviceBuffer.from_numpy(wk), norm_eps=1e-6,
                       rope=rope is not None and DeviceBuffer.from_numpy(rope) or None, positions=pos is not None and i32(pos) or None, x_stride=stride, out_stride=stride if in_place else 0)
  rot = rope[pos] if r else None
  got = get(out, (rows, h + 2 * hk + 1 if in_place else h + hk, d), ot)
  for a, b, w in ((0, h, wq), (h, h + hk, wk)): close_rows(got[:, a:b], ref.rotate(ref.head_norm(xv[:, a:b], w, 1e-6), rot), reach_of(xv[:, a:b], w, 1e-6, rot), ot, str(a))
  if in_place: assert (got[:, h + hk:] == xv[:, h + hk:]).all()


def test_head_norm_rope_position_outside_the_table():
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer
  x, xv = put(np.ones((3, 2, 32)), "float32")
  status()
  paged.head_norm_rope(x, x, 3, 1, 1, 32, rope=DeviceBuffer.from_numpy(cos_sin(4, 32)), positions=i32([-1, 0, 4]))
  got = get(x, (3, 64), "float32")
  assert (got[1] == 1).all() and not got[0].any() and not got[2].any() and status() == 2


# ---- attention ----
# Tolerance.  Scores: products of `dim` values added in 32 bits, in an order of the kernel's choice, tensor cores cutting where others round: a walk of dim steps of at most 2^-23 of the sum of
# magnitudes, 4 sqrt(dim) of them; a step of a score moves its probability by that much (and the others' sum by no more): twice that, of sum p |v|.  The exponential and its argument: 2^-21.  The sum over n
# keys: 4 sqrt(n) 2^-23.  Half a step of the output.  Kernels that take probabilities to the tensor core in the 16 bits of the cache (16-bit queries) lose half a step of that too.
def close_attention(got, want, weight, reach, dim, keys, q_type, out_type, what):
  tol = weight * (2 * 4 * dim ** 0.5 * 2.0 ** -23 * reach[..., None] + 2.0 ** -21 + 4 * keys ** 0.5 * 2.0 ** -23)
  if q_type != "float32": tol = tol + weight * EPS[q_type] / 2
  tol = tol + EPS[out_type] / 2 * (np.abs(want) + tol) + TINY[out_type]
  bad = ~(np.abs(got - want) <= tol)
  assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, worst {np.max(np.abs(got - want) / np.maximum(tol, 1e-300)):.2f} tolerances, first at {np.argwhere(bad)[0]}"


def attend(seqs, h, hk, d, ps, qt, ct, ot=None, lay="head-major", seed=0, scale=0.0, pad=2, spread=1.0, poison=True, bounds=None, tables=None, stream=None):
  """One call against the oracle.  poison: everything in the pools that belongs to no position of a sequence is NaN."""
  from tinygrad_b200 import paged
  ot = ot or qt
  rng = np.random.default_rng(seed)
  new, length = [n for n, _ in seqs], [l for _, l in seqs]
  off, n = np.concatenate([[0], np.cumsum(new)]), sum(new)
  t, n_pages = table(rng, length, ps)
  strides, size = layout(lay, n_pages, hk, ps, d)
  pools = []
  for _ in "kv":
    flat = np.full(size, np.nan if poison else 0.0, np.float32)
    view = in_layout(flat, strides, n_pages, hk, ps, d)
    for s, l in enumerate(length):
      p = np.arange(l)
      view[t[s][p // ps], :, p % ps] = rng.standard_normal((l, hk, d))
    buf, val = put(flat, ct)
    pools.append((buf, in_layout(val, strides, n_pages, hk, ps, d)))
  q, qv = put(rng.standard_normal((n + pad, h, d)) * spread, qt)
  out, _ = put(np.full((n + pad, h, d), 3.0), ot)
  status()
  cache = paged.PagedCache(n_pages, ps, hk, d, ct, k=pools[0][0], v=pools[1][0], strides=strides)
  most_new, most_len = bounds or (max(new), max(length))
  batch = paged.PagedBatch(i32(off), i32(length), i32(t), n_rows=n + pad, max_new=most_new, max_len=most_len)
  want, weight, reach = ref.attention(qv[:n], pools[0][1], pools[1][1], off, length, t, ps, scale or d ** -0.5)
  for again in range(2):      # (the second call finds the workspace as the first has left it)
    paged.attention(cache, batch, q, out, h, qt, out_dtype=ot, scale=scale, stream=stream)
    if stream is not None: stream.synchronize()
    got = get(out, (n + pad, h, d), ot)
    close_attention(got[:n], want, weight, reach, d, max(length), qt, ot, f"call {again}")
    assert (got[n:] == 3).all(), "rows behind the last sequence are left as they were"
  assert status() == 0
  return got[:n]


ATTEND = [   # seqs' (new, length), heads, KV heads, dim, page size, types of q / pages / out
  ([(1, 1)], 4, 2, 64, 16, "float32", "float16", None),
  ([(1, 513)], 32, 8, 128, 16, "float32", "float16", None),
  ([(1, 2000), (1, 3), (1, 64), (1, 1025)], 28, 4, 128, 64, "float32", "float16", None),
  ([(1, 700), (0, 50), (1, 701)], 8, 8, 128, 32, "float16", "float16", None),
  ([(3, 300), (4, 4), (2, 129)], 7, 1, 64, 16, "bfloat16", "bfloat16", None),
  ([(40, 40), (1, 100), (129, 260)], 4, 2, 128, 16, "float32", "float16", "float16"),
  ([(70, 333)], 6, 3, 32, 5, "float32", "bfloat16", None),
  ([(17, 17), (5, 90)], 3, 1, 16, 1, "float16", "bfloat16", "float32"),
  ([(65, 200), (3, 1500)], 4, 1, 64, 100, "float32", "float32", None),
  ([(1, 4097)], 4, 4, 128, 128, "float32", "float32", None),
  ([(200, 700)], 8, 2, 128, 128, "float16", "float16", None),
  ([(257, 257), (130, 1000), (1, 900)], 8, 2, 64, 32, "bfloat16", "bfloat16", None),
  ([(129, 129)], 5, 5, 128, 8, "float16", "float16", None),
  ([(300, 5000)], 4, 1, 128, 16, "float16", "float16", None),
  ([(90, 4000)], 16, 1, 64, 256, "float16", "float16", "float32"),
  ([(150, 150), (2, 60)], 7, 1, 128, 64, "bfloat16", "bfloat16", "float16"),
  ([(1, 300), (3, 90)], 40, 1, 64, 32, "float32", "float16", None),                                     # more heads to a key head than a tile of 16 rows has
  ([(1 + i % 3, 20 + 7 * i) for i in range(70)], 4, 2, 64, 16, "float16", "float16", None),             # more sequences than a warp has lanes
  ([(i % 2 * (1 + i), 5 + 9 * i) for i in range(40)], 2, 1, 128, 16, "float32", "float16", None),       # many without new tokens, few and many rows in one batch
  ([(260, 900), (1, 3000), (0, 7), (33, 33)], 8, 8, 128, 16, "float32", "float16", "float16"),
]


@pytest.mark.parametrize("lay", ["head-major", "slot-major", "loose"])
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention(case, lay):
  need_gpu()
  seqs, h, hk, d, ps, qt, ct, ot = ATTEND[case]
  attend(seqs, h, hk, d, ps, qt, ct, ot, lay, seed=case)


@pytest.mark.parametrize("qt,ct", [("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16"), ("float32", "bfloat16")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("seqs", [[(1, 900), (1, 17)], [(200, 900), (9, 9)]], ids=["tokens", "chunks"])
def test_attention_with_peaked_scores_and_a_scale(qt, ct, d, seqs):
  """Scores some hundred apart: the running maximum moves, most probabilities vanish."""
  need_gpu()
  attend(seqs, 4, 2, d, 16, qt, ct, seed=d, spread=20.0)
  attend(seqs, 4, 2, d, 16, qt, ct, seed=d, scale=0.03)


@pytest.mark.parametrize("qt,ct", [("float32", "float16"), ("float16", "float16"), ("float32", "float32")])
def test_rows_without_a_position(qt, ct):
  """length below the number of new rows: the first of them stand before position 0, see nothing and get zeros."""
  need_gpu()
  got = attend([(5, 2), (3, 0), (150, 20), (1, 0)], 4, 2, 64, 16, qt, ct, seed=3)
  assert not got[:3].any() and got[3].any() and not got[5:8].any() and not got[8:138].any() and got[138].any() and not got[158].any()


@pytest.mark.parametrize("qt,ct", [("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16"), ("float32", "float32")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,length,at", [(4, 100, 98), (200, 400, 300), (130, 130, 1), (130, 140, 139)])
def test_values_behind_a_rows_position_are_not_read_into_it(qt, ct, d, new, length, at):
  """A later token's key and value are NaN or infinite: rows before it are what they were, rows from it on are not finite (NaN)."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(at)
  h, hk, ps = 4, 2, 16
  t, n_pages = table(rng, [length], ps)
  outs = []
  k, v, q = rng.standard_normal((n_pages, hk, ps, d)), rng.standard_normal((n_pages, hk, ps, d)), rng.standard_normal((new, h, d))
  for bad in (None, (np.nan, np.nan), (0.5, np.nan), (0.5, np.inf)):
    if bad is not None:
      k[t[0, at // ps], :, at % ps], v[t[0, at // ps], :, at % ps, 5] = bad[0], bad[1]
    cache = paged.PagedCache(n_pages, ps, hk, d, ct, k=put(k, ct)[0], v=put(v, ct)[0])
    batch = paged.PagedBatch(i32([0, new]), i32([length]), i32(t), n_rows=new, max_new=new, max_len=length)
    out = put(np.zeros((new, h, d)), qt)[0]
    paged.attention(cache, batch, put(q, qt)[0], out, h, qt)
    outs.append(get(out, (new, h, d), qt))
  sees = np.arange(new) + length - new >= at
  for bad in outs[1:]:
    assert (bad[~sees] == outs[0][~sees]).all()
    assert not np.isfinite(bad[sees][..., 5]).any()
  assert np.isfinite(outs[2][sees][..., 6]).all() and np.isfinite(outs[3][sees][..., 6]).all()


def test_attention_where_the_tables_are_wrong():
  """Pages that do not exist read as zeros; what lies past a bound is not attended, or not computed; status 2 each time."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(8)
  h, hk, d, ps, n_pages = 4, 2, 64, 16, 7
  for qt, ct, new in (("float32", "float16", 1), ("float16", "float16", 40), ("float32", "float32", 3), ("float16", "float16", 200)):
    length = 210
    (k, kv), (v, vv), (q, qv) = (put(rng.standard_normal(s), t) for s, t in (((n_pages, hk, ps, d), ct), ((n_pages, hk, ps, d), ct), ((new, h, d), qt)))
    t = rng.integers(0, n_pages, (1, 14)).astype(np.int32)      # (the same page twice is fine)
    t[0, [2, 9]] = -1, n_pages
    cache = paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v)
    out = put(np.full((new, h, d), 9.0), qt)[0]
    status()
    paged.attention(cache, paged.PagedBatch(i32([0, new]), i32([length]), i32(t), n_rows=new, max_new=new, max_len=length), q, out, h, qt)
    want, weight, reach = ref.attention(qv, kv, vv, [0, new], [length], t, ps, d ** -0.5)
    close_attention(get(out, (new, h, d), qt), want, weight, reach, d, length, qt, qt, "pages")
    assert status() == 2
    # a length past the bound: keys 0 .. max_len - 1, every row at its own position
    t[0, [2, 9]] = 0
    paged.attention(cache, paged.PagedBatch(i32([0, new]), i32([length]), i32(t), n_rows=new, max_new=new, max_len=150), q, out, h, qt)
    got = get(out, (new, h, d), qt)
    keep = [i for i in range(new) if length - new + i < 150]
    want, weight, reach = ref.attention(qv, kv, vv, [0, new], [length], t, ps, d ** -0.5)
    if keep: close_attention(got[keep], want[keep], weight[keep], reach[keep], d, length, qt, qt, "rows below the bound")
    want, weight, reach = ref.attention(qv[-1:], kv, vv, [0, 1], [150], t, ps, d ** -0.5)
    close_attention(got[-1:], want, weight, reach, d, length, qt, qt, "the last row")
    assert status() == 2
    if new > 1:      # more rows than the bound
      out = put(np.full((new, h, d), 9.0), qt)[0]
      paged.attention(cache, paged.PagedBatch(i32([0, new]), i32([length]), i32(t), n_rows=new, max_new=new - 1, max_len=length), q, out, h, qt)
      got = get(out, (new, h, d), qt)
      assert (got[-1] == 9).all() and not (got[-2] == 9).any() and status() == 2


@pytest.mark.parametrize("ct", ["float16", "float32"])
def test_attention_of_rows_that_go_back(ct):
  """row_off 0, 3, 1, 4: sequences overlap.  Status 2, nothing outside the rows is written, and the work stays what the bounds allow."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(21)
  (k, _), (v, _), (q, _) = (put(rng.standard_normal(s), t) for s, t in (((4, 2, 16, 64), ct), ((4, 2, 16, 64), ct), ((5, 4, 64), "float32")))
  out = put(np.full((5, 4, 64), 9.0), "float32")[0]
  batch = paged.PagedBatch(i32([0, 3, 1, 4]), i32([40, 50, 60]), i32(rng.integers(0, 4, (3, 4))), n_rows=5, max_new=3, max_len=60)
  status()
  paged.attention(paged.PagedCache(4, 16, 2, 64, ct, k=k, v=v), batch, q, out, 4)
  assert (get(out, (5, 4, 64), "float32")[4] == 9).all() and status() == 2


def test_attention_of_views():
  """Rows of torch tensors that lie apart, in and out."""
  need_gpu()
  import torch
  from tinygrad_b200 import paged
  rng = np.random.default_rng(22)
  n, h, hk, d, length = 3, 4, 2, 64, 45
  (k, kv), (v, vv) = (put(rng.standard_normal((4, hk, 16, d)), "float16") for _ in range(2))
  q, out = torch.from_numpy(rng.standard_normal((n, h * d + 40))).half().cuda()[:, 40:], torch.full((n, h * d + 8), 9.0, device="cuda")[:, :h * d]
  t = rng.integers(0, 4, (1, 3)).astype(np.int32)
  cache, batch = paged.PagedCache(4, 16, hk, d, "float16", k=k, v=v), paged.PagedBatch(i32([0, n]), i32([length]), i32(t), n_rows=n, max_new=n, max_len=length)
  torch.cuda.synchronize()
  paged.attention(cache, batch, q, out, h, "float16", "float32", q_stride=h * d + 40, out_stride=h * d + 8)
  from tinygrad_b200 import runtime
  runtime.synchronize()
  want, weight, reach = ref.attention(q.cpu().double().numpy().reshape(n, h, d), kv, vv, [0, n], [length], t, 16, d ** -0.5)
  close_attention(out.cpu().double().numpy().reshape(n, h, d), want, weight, reach, d, length, "float16", "float32", "views")
  assert (out._base[:, h * d:] == 9).all()


def test_attention_gives_the_same_bits_again():
  need_gpu()
  for args in (([(1, 3000), (1, 70)], 8, 2, 128, 16, "float32", "float16"), ([(300, 4000)], 8, 2, 128, 16, "float16", "float16"), ([(3, 2500)], 4, 2, 64, 16, "bfloat16", "bfloat16")):
    a, b = attend(*args, seed=1), attend(*args, seed=1)
    assert (a == b).all()


@pytest.mark.parametrize("qt,ct", [("float16", "float16"), ("bfloat16", "bfloat16"), ("float32", "float16")])
@pytest.mark.parametrize("seqs", [[(1, 200), (2, 33)], [(140, 300), (1, 90)]], ids=["tokens", "chunks"])
def test_attention_of_rows_on_odd_boundaries(qt, ct, seqs):
  """Queries and outputs one element off, with strides that are no multiple of 16 bytes: the same values as on whole boundaries."""
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer
  rng = np.random.default_rng(3)
  h, hk, d, ps = 4, 2, 64, 16
  new, length = [n for n, _ in seqs], [l for _, l in seqs]
  off, n = np.concatenate([[0], np.cumsum(new)]), sum(new)
  t, n_pages = table(rng, length, ps)
  (k, _), (v, _) = (put(rng.standard_normal((n_pages, hk, ps, d)), ct) for _ in "kv")
  x = rng.standard_normal((n, h * d))
  cache = paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v)
  batch = paged.PagedBatch(i32(off), i32(length), i32(t), n_rows=n, max_new=max(new), max_len=max(length))
  q, out = put(x, qt)[0], put(np.zeros((n, h * d)), qt)[0]
  paged.attention(cache, batch, q, out, h, qt)
  size, stride = 4 if qt == "float32" else 2, h * d + 3
  wide = np.zeros((n * stride + 1,))
  np.lib.stride_tricks.as_strided(wide[1:], (n, h * d), (8 * stride, 8))[:] = x
  q2, out2 = put(wide, qt)[0], put(np.full(n * stride + 1, 5.0), qt)[0]
  paged.attention(cache, batch, q2.ptr + size, out2.ptr + size, h, qt, q_stride=stride, out_stride=stride)
  got = get(out2, (n * stride + 1,), qt)
  rows = np.lib.stride_tricks.as_strided(got[1:], (n, h * d), (8 * stride, 8))
  assert (rows == get(out, (n, h * d), qt)).all()
  rows[:] = 5
  assert (got == 5).all(), "what lies between the rows is as it was"


def test_one_workspace_for_calls_of_any_shape():
  """A batch's workspace serves one call after the other, of any cache and number of heads: no call finds what another has left."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(13)
  new, length = [1, 130, 2], [3000, 1500, 700]
  off, n = np.concatenate([[0], np.cumsum(new)]), sum(new)
  calls = []
  t, n_pages = table(rng, length, 16)
  tables = [i32(off), i32(length), i32(t)]
  for h, hk, d, qt, ct in ((8, 2, 128, "float16", "float16"), (4, 4, 64, "float32", "float32"), (28, 4, 128, "float32", "float16"), (4, 1, 32, "bfloat16", "bfloat16"), (2, 1, 64, "float16", "float16")):
    (k, _), (v, _) = (put(rng.standard_normal((n_pages, hk, 16, d)), ct) for _ in "kv")
    q, out = put(rng.standard_normal((n, h, d)), qt)[0], put(np.zeros((n, h, d)), qt)[0]
    calls.append((paged.PagedCache(n_pages, 16, hk, d, ct, k=k, v=v), q, out, h, d, qt))
  alone = []
  for cache, q, out, h, d, qt in calls:
    paged.attention(cache, paged.PagedBatch(*tables, n_rows=n, max_new=130, max_len=3000), q, out, h, qt)
    alone.append(get(out, (n, h, d), qt))
  batch = paged.PagedBatch(*tables, n_rows=n, max_new=130, max_len=3000)
  for _ in range(2):
    for (cache, q, out, h, d, qt), want in zip(calls, alone):
      out.zero_()
      paged.attention(cache, batch, q, out, h, qt)
      assert (get(out, (n, h, d), qt) == want).all(), (h, d, qt)
  assert status() == 0


def test_two_streams_at_once():
  """A batch (and workspace) for each stream: calls that run at the same time do not disturb each other."""
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import Stream
  rng = np.random.default_rng(14)
  h, hk, d, ps, new, length = 8, 2, 128, 16, [1, 200], [20000, 4000]
  t, n_pages = table(rng, length, ps)
  (k, _), (v, _) = (put(rng.standard_normal((n_pages, hk, ps, d)), "float16") for _ in "kv")
  cache = paged.PagedCache(n_pages, ps, hk, d, k=k, v=v)
  q = [put(rng.standard_normal((201, h, d)), "float16")[0] for _ in range(2)]
  out = [put(np.zeros((201, h, d)), "float16")[0] for _ in range(2)]
  batches = [paged.PagedBatch(i32([0, 1, 201]), i32(length), i32(t), n_rows=201, max_new=200, max_len=20000) for _ in range(2)]
  want = []
  for i in range(2):
    paged.attention(cache, batches[i], q[i], out[i], h, "float16")
    want.append(get(out[i], (201, h, d), "float16"))
    out[i].zero_()
  streams = [Stream(), Stream()]
  for _ in range(10):
    for i in range(2): paged.attention(cache, batches[i], q[i], out[i], h, "float16", stream=streams[i])
  for s in streams: s.synchronize()
  for i in range(2): assert (get(out[i], (201, h, d), "float16") == want[i]).all()


def test_pools_past_32_bits():
  """Pages 2^28 elements apart, ten of them: offsets pass 2^31 elements and 2^32 bytes, for appending and for every attention kernel."""
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer
  rng = np.random.default_rng(15)
  h, hk, d, ps, apart = 4, 2, 64, 16, 1 << 28
  size = 9 * apart + hk * ps * d
  k, v = DeviceBuffer(2 * size), DeviceBuffer(2 * size)
  far = paged.PagedCache(10, ps, hk, d, k=k, v=v, strides=(apart, ps * d, d))
  near = paged.PagedCache(10, ps, hk, d)
  x, _ = put(rng.standard_normal((150, h + 2 * hk, d)), "float16")
  pages = i32(rng.permutation(10)[None])
  outs = []
  for cache in (near, far):
    q, out = put(np.zeros((150, h, d)), "float16")[0], put(np.zeros((150, h, d)), "float16")[0]
    batch = paged.PagedBatch(i32([0, 150]), i32([150]), pages, n_rows=150, max_new=150, max_len=150)
    paged.append(cache, batch, x, q, h, "float16")
    paged.attention(cache, batch, q, out, h, "float16")
    one = put(np.zeros((1, h, d)), "float16")[0]
    paged.attention(cache, paged.PagedBatch(i32([0, 1]), i32([150]), pages, n_rows=1, max_new=1, max_len=150), q, one, h, "float16")
    outs.append((get(out, (150, h, d), "float16"), get(one, (1, h, d), "float16")))
  assert (outs[0][0] == outs[1][0]).all() and (outs[0][1] == outs[1][1]).all() and outs[0][0].any()
  assert status() == 0


@pytest.mark.parametrize("qt,ct", [("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16"), ("float32", "float32")])
@pytest.mark.parametrize("new", [2, 150])
def test_queries_that_are_not_finite(qt, ct, new):
  """A row of queries that is NaN or infinite gives a row of NaN; the others are what they were.  A row of zeros gives the mean of the values."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(new)
  h, hk, d, ps, length = 2, 1, 64, 16, 200
  t, n_pages = table(rng, [length], ps)
  (k, _), (v, vv) = (put(rng.standard_normal((n_pages, hk, ps, d)), ct) for _ in "kv")
  cache = paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v)
  batch = paged.PagedBatch(i32([0, new]), i32([length]), i32(t), n_rows=new, max_new=new, max_len=length)
  x = rng.standard_normal((new, h, d))
  x[new - 1, 1] = 0
  outs = []
  for bad in (None, np.nan, np.inf):
    if bad is not None: x[0, 0, 3] = bad
    out = put(np.zeros((new, h, d)), qt)[0]
    paged.attention(cache, batch, put(x, qt)[0], out, h, qt)
    outs.append(get(out, (new, h, d), qt))
  for got in outs[1:]:
    assert np.isnan(got[0, 0]).all()
    got[0, 0] = outs[0][0, 0]
    assert (got == outs[0]).all()
  mean = ref.gather(vv, t[0], length, ps)[0].mean(0)
  spread = np.abs(ref.gather(vv, t[0], length, ps)[0]).mean(0)
  assert (np.abs(outs[0][new - 1, 1] - mean) <= spread * (2.0 ** -21 + 4 * length ** 0.5 * 2.0 ** -23 + EPS[qt]) + EPS[qt] / 2 * np.abs(mean)).all()


def test_append_of_more_sequences_than_a_warp_has_lanes():
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(16)
  h, hk, d, ps = 2, 1, 32, 8
  new = [int(x) for x in rng.integers(0, 4, 100)]
  length = [n + int(x) for n, x in zip(new, rng.integers(0, 30, 100))]
  off, n = np.concatenate([[0], np.cumsum(new)]), sum(new)
  t, n_pages = table(rng, length, ps)
  x, xv = put(rng.standard_normal((n, h + 2 * hk, d)), "float32")
  cache = paged.PagedCache(n_pages, ps, hk, d, "float32")
  q = put(np.zeros((n, h, d)), "float32")[0]
  paged.append(cache, paged.PagedBatch(i32(off), i32(length), i32(t), n_rows=n, max_new=3, max_len=max(length)), x, q, h)
  assert (get(q, (n, h, d), "float32") == xv[:, :h]).all()
  k = get(cache.k, (n_pages, hk, ps, d), "float32")
  for row, (s, p) in enumerate(ref.rows_of(off, length)): assert (k[t[s][p // ps], :, p % ps] == xv[row, h:h + hk]).all()
  assert (k != 0).any(-1).sum() == n


def test_nothing_to_do():
  need_gpu()
  from tinygrad_b200 import paged
  cache = paged.PagedCache(2, 16, 1, 64)
  x, _ = put(np.ones((4, 3, 64)), "float32")
  out, _ = put(np.full((4, 1, 64), 2.0), "float32")
  for off, length in (([0, 0], [0]), ([0, 0, 0], [5, 0])):
    batch = paged.PagedBatch(i32(off), i32(length), i32(np.zeros((len(length), 1))), n_rows=4, max_new=1, max_len=16)
    paged.append(cache, batch, x, out, 1)
    paged.attention(cache, batch, x, out, 1)
  paged.attention(cache, paged.PagedBatch(i32([0]), i32(np.zeros(0)), i32(np.zeros((0, 1))), n_rows=0, max_new=0, max_len=0), x, out, 1)
  paged.head_norm_rope(x, out, 0, 1, 0, 64)
  assert (get(out, (4, 64), "float32") == 2).all() and status() == 0


# ---- as a serving program uses them ----
@pytest.mark.parametrize("xt,ct", [("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")])
def test_prompts_and_tokens_of_two_sequences(xt, ct):
  """Two sequences: a prompt each in chunks of different sizes, then single tokens in a captured graph whose lengths and pages change on the device; every row against causal attention over the whole
  sequence."""
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer, Graph, Stream
  rng = np.random.default_rng(4)
  h, hk, d, ps, total = 8, 2, 64, 16, (150, 61)
  steps = [(40, 0), (90, 33), (1, 20)] + [(1, 1)] * 8
  stream = Stream()
  cache = paged.PagedCache(20, ps, hk, d, ct)
  x = [rng.standard_normal((n, h + 2 * hk, d)) for n in total]
  w = rng.uniform(0.5, 1.5, (2, d)).astype(np.float16)
  rope = cos_sin(200, d)
  rope_d, wq, wk = DeviceBuffer.from_numpy(rope), DeviceBuffer.from_numpy(w[0]), DeviceBuffer.from_numpy(w[1])
  pages = rng.permutation(20).reshape(2, 10).astype(np.int32)
  at, got, graph = [0, 0], [[], []], None
  one = None
  for new in steps:
    rows = np.concatenate([x[s][at[s]:at[s] + n] for s, n in enumerate(new)])
    at = [a + n for a, n in zip(at, new)]
    off = np.array([0, new[0], sum(new)], np.int32)
    if new == (1, 1):
      if one is None:
        one = [put(rows, xt)[0], put(rows[:, :h], xt)[0], put(rows[:, :h], xt)[0], i32(off), i32(at), i32(np.zeros((2, 10)))]
        batch = paged.PagedBatch(*one[3:], n_rows=2, max_new=1, max_len=200)
        batch.reserve(cache, h, xt)
        graph = Graph(stream)
        with graph:
          paged.append(cache, batch, one[0], one[1], h, xt, rope=rope_d, q_norm=wq, k_norm=wk, norm_eps=1e-6, stream=stream)
          paged.attention(cache, batch, one[1], one[2], h, xt, flags=1, stream=stream)
      xb = rows.astype(xt) if xt != "bfloat16" else ref.bf16_bits(rows.astype(np.float32))
      one[0].copy_from(xb), one[4].copy_from(np.array(at, np.int32)), one[5].copy_from(pages)
      graph.launch()
      stream.synchronize()
      out = get(one[2], (2, h, d), xt)
    else:
      xb, q, o = put(rows, xt)[0], put(rows[:, :h], xt)[0], put(rows[:, :h], xt)[0]
      batch = paged.PagedBatch(i32(off), i32(at), i32(pages), n_rows=sum(new), max_new=max(new), max_len=max(at))
      paged.append(cache, batch, xb, q, h, xt, rope=rope_d, q_norm=wq, k_norm=wk, norm_eps=1e-6, stream=stream)
      paged.attention(cache, batch, q, o, h, xt, stream=stream)
      stream.synchronize()
      out = get(o, (sum(new), h, d), xt)
    got[0].append(out[:new[0]]), got[1].append(out[new[0]:])
  k = get(cache.k, (20, hk, ps, d), ct), get(cache.v, (20, hk, ps, d), ct)
  for s in range(2):
    n = at[s]
    xs = put(x[s][:n], xt)[1]
    q = ref.rotate(ref.head_norm(xs[:, :h], w[0], 1e-6), rope[:n])
    qd = put(q, xt)[1]                       # rounded once by append
    want, weight, reach = ref.attention(qd, *k, [0, n], [n], pages[s:s + 1], ps, d ** -0.5)
    # append's q may be rounded the other way where it is half way between two values: a step of q moves a score by EPS / 2 of its reach
    slack = weight * 2 * EPS[xt] / 2 * reach[..., None]
    tol_got = np.concatenate(got[s])
    err = np.abs(tol_got - want)
    tol = weight * (2 * 4 * d ** 0.5 * 2.0 ** -23 * reach[..., None] + 2.0 ** -21 + 4 * n ** 0.5 * 2.0 ** -23 + (EPS[xt] / 2 if xt != "float32" else 0)) + slack
    assert (err <= tol + EPS[xt] / 2 * (np.abs(want) + tol) + TINY[xt]).all(), s
  assert status() == 0


def test_against_the_contiguous_cache():
  """The same prompt through b200q_attn_prefill and through pages: both within their tolerance of each other."""
  need_gpu()
  from tinygrad_b200 import _lib, paged
  from tinygrad_b200.runtime import DeviceBuffer
  rng = np.random.default_rng(6)
  h, hk, d, n, ctx, ps = 8, 2, 128, 90, 128, 16
  x = rng.standard_normal((n, (h + 2 * hk) * d)).astype(np.float32)
  rope = cos_sin(ctx, d)
  xb, rb = DeviceBuffer.from_numpy(x), DeviceBuffer.from_numpy(rope)
  k, v = (DeviceBuffer.empty((hk, ctx, d), np.float16, zero=True) for _ in "kv")
  q, out = DeviceBuffer.empty((n, h * d), np.float32), DeviceBuffer.empty((n, h * d), np.float32)
  _lib.check(_lib.load().b200q_attn_prefill(xb.ptr, k.ptr, v.ptr, _lib.F16, rb.ptr, 0, n, h, hk, d, d, ctx, q.ptr, out.ptr, _lib.F32, None))
  want = out.numpy()
  cache = paged.PagedCache(8, ps, hk, d)
  pages = rng.permutation(8).astype(np.int32)[None]
  batch = paged.PagedBatch(i32([0, n]), i32([n]), i32(pages), n_rows=n, max_new=n, max_len=n)
  paged.append(cache, batch, xb, q, h, rope=rb)
  paged.attention(cache, batch, q, out, h)
  kp = cache.k.numpy((8, hk, ps, d), np.float16)[pages[0]].transpose(1, 0, 2, 3).reshape(hk, ctx, d)
  # a c - b s in 32 bits with one of the products rounded or the other: two values within 2^-23 (|a| + |b|) of each other, which may lie on either side of a border between two
  # fp16 values.  They are rounded to neighbours then: a step of the larger one apart, 2^-10 of it at most
  kc = k.numpy()[:, :n].astype(np.float64)
  assert (np.abs(kp[:, :n].astype(np.float64) - kc) <= EPS["float16"] * np.abs(kc) + 2 * TINY["float16"]).all()
  np.testing.assert_allclose(out.numpy(), want, rtol=0, atol=2e-5)


@pytest.mark.parametrize("qt,ct,d,seqs", [("float16", "float16", 128, [(200, 700), (1, 300), (9, 60)]), ("bfloat16", "bfloat16", 64, [(90, 3000), (2, 40)]), ("float32", "float16", 128, [(40, 2000)])],
                         ids=["both kernels", "keys in parts beside tokens", "keys in parts"])
def test_captured_chunks(qt, ct, d, seqs):
  """A call of several kernels in a graph: the eager call's bits, and those of other tables after they have changed on the device."""
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import Graph, Stream
  rng = np.random.default_rng(31)
  h, hk, ps = 8, 2, 16
  new, length = [n for n, _ in seqs], [l for _, l in seqs]
  off, n = np.concatenate([[0], np.cumsum(new)]), sum(new)
  t, n_pages = table(rng, length, ps)
  t = np.maximum(t, 0)
  (k, _), (v, _), (q, _) = (put(rng.standard_normal(s), c) for s, c in (((n_pages, hk, ps, d), ct), ((n_pages, hk, ps, d), ct), ((n, h, d), qt)))
  cache, lens, pages, stream = paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v), i32(length), i32(t), Stream()
  batch, out = paged.PagedBatch(i32(off), lens, pages, n_rows=n, max_new=max(new), max_len=max(length)), put(np.zeros((n, h, d)), qt)[0]
  status()
  batch.reserve(cache, h)
  graph = Graph(stream)
  with graph:
    paged.attention(cache, batch, q, out, h, qt, stream=stream)
  for now in (length, [max(m, l - 70) for m, l in seqs]):
    lens.copy_from(np.asarray(now, np.int32))
    pages.copy_from(np.ascontiguousarray(t[:, ::-1] if now is not length else t))
    paged.attention(cache, batch, q, out, h, qt)
    want = out.numpy((n, h, d), np.uint32 if qt == "float32" else np.uint16)
    for _ in range(3):
      out.copy_from(np.zeros((n, h, d), want.dtype))
      graph.launch()
      stream.synchronize()
      assert (out.numpy((n, h, d), want.dtype) == want).all()
  assert status() == 0


@pytest.mark.parametrize("seqs", [[(1, 300)] * 5, [(150, 400), (3, 90), (1, 1200)], [(70, 2500)]], ids=["tokens", "both kernels", "keys in parts"])
def test_a_chain_of_dependent_launches(seqs):
  """append and attention in turn, each told that the launch before it is the library's own: bits of the calls without that."""
  need_gpu()
  from tinygrad_b200 import _lib, paged
  from tinygrad_b200.runtime import synchronize
  rng = np.random.default_rng(32)
  h, hk, d, ps, layers = 8, 2, 64, 16, 6
  new, length = [n for n, _ in seqs], [l for _, l in seqs]
  off, n = np.concatenate([[0], np.cumsum(new)]), sum(new)
  t, n_pages = table(rng, length, ps)
  old = rng.standard_normal((2, layers, n_pages, hk, ps, d))
  xs = [put(rng.standard_normal((n, (h + 2 * hk) * d)), "float16")[0] for _ in range(layers)]
  batch = paged.PagedBatch(i32(off), i32(length), i32(t), n_rows=n, max_new=max(new), max_len=max(length))
  got = []
  for flags in (0, _lib.FLAG_PDL):
    caches = [paged.PagedCache(n_pages, ps, hk, d, "float16", k=put(old[0, i], "float16")[0], v=put(old[1, i], "float16")[0]) for i in range(layers)]
    q, outs = put(np.zeros((n, h * d)), "float16")[0], [put(np.zeros((n, h * d)), "float16")[0] for _ in range(layers)]
    batch.reserve(caches[0], h)
    synchronize()
    for i in range(layers):      # (q and the workspace are every layer's)
      paged.append(caches[i], batch, xs[i], q, h, "float16", flags=flags if i else 0)
      paged.attention(caches[i], batch, q, outs[i], h, "float16", flags=flags)
    got.append([o.numpy((n, h * d), np.uint16) for o in outs])
  for a, b in zip(*got): assert (a == b).all()
  assert any(a.any() for a in got[0])


@pytest.mark.parametrize("qt,ct", [("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "bfloat16"), ("float32", "float32")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,length", [(2, 100), (2, 3000), (200, 400), (200, 3000)], ids=["tokens", "tokens, keys in parts", "chunk", "chunk, keys in parts"])
def test_scores_of_minus_infinity(qt, ct, d, new, length):
  """A row whose scores are all minus infinity gets zeros, one with some such scores the others' mean: keys of weight 0 leave nothing behind, however large their values are.  fp16: an infinite query
  or key gives such a score; the wider types: 2^100 times -2^100."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(new + length)
  h, hk, ps = 4, 2, 16
  t, n_pages = table(rng, [length], ps)
  out_of = np.zeros(length, bool)          # keys that no row gives a weight: the first tiles whole, some of the rest
  out_of[:min(256, length // 3)] = True
  out_of |= rng.random(length) < 0.3
  big, low = (np.inf, -np.inf) if ct == "float16" else (2.0 ** 100, -2.0 ** 100)
  k, v, q = rng.standard_normal((length, hk, d)), rng.standard_normal((length, hk, d)), rng.standard_normal((new, h, d))
  k[:, :, 0], q[:, :, 0] = (-1.0 if ct == "float16" else low), 0.0
  k[:, :, 1], q[:, :, 1] = np.where(out_of, low, 0.0)[:, None], (1.0 if ct == "float16" else big)
  v[out_of, :, 3] = 60000.0 if ct == "float16" else 2.0 ** 126
  none = [(0, 0), (new // 2, 3), (new - 1, 1)]
  for r, j in none: q[r, j, 0] = big
  pools = []
  for x in (k, v):
    pool = np.zeros((n_pages, hk, ps, d), np.float32)
    p = np.arange(length)
    pool[t[0][p // ps], :, p % ps] = x
    pools.append(put(pool, ct))
  kv = [ref.gather(val, t[0], length, ps) for _, val in pools]
  qb, qv = put(q, qt)
  out = put(np.full((new, h, d), 3.0), qt)[0]
  status()
  paged.attention(paged.PagedCache(n_pages, ps, hk, d, ct, k=pools[0][0], v=pools[1][0]), paged.PagedBatch(i32([0, new]), i32([length]), i32(t), n_rows=new, max_new=new, max_len=length), qb, out, h, qt)
  got = get(out, (new, h, d), qt)
  assert status() == 0
  want, weight, reach = np.zeros((new, h, d)), np.zeros((new, h, d)), np.zeros((new, h))
  for r in range(new):
    sees = ~out_of & (np.arange(length) <= length - new + r)
    for j in range(h):
      if (r, j) in none or not sees.any():
        assert not got[r, j].any(), (r, j)
        continue
      kk, vv = kv[0][j // 2][sees, 2:], kv[1][j // 2][sees]
      s = kk @ qv[r, j, 2:] * d ** -0.5
      e = np.exp(s - s.max())
      e /= e.sum()
      want[r, j], weight[r, j], reach[r, j] = e @ vv, e @ np.abs(vv), (np.abs(kk) @ np.abs(qv[r, j, 2:])).max() * d ** -0.5
  close_attention(got, want, weight, reach, d, length, qt, qt, "rows with some scores of minus infinity")


@pytest.mark.parametrize("qt,ct", [("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16"), ("float32", "bfloat16")])
@pytest.mark.parametrize("new,length", [(2, 300), (150, 400), (150, 3000)])
def test_queries_that_are_not_finite_in_wide_heads(qt, ct, new, length):
  """Heads of 128, keys whole and in parts: a row of queries that is NaN or infinite gives a row of NaN, the others keep their bits."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(new)
  h, hk, d, ps = 2, 1, 128, 16
  t, n_pages = table(rng, [length], ps)
  (k, _), (v, _) = (put(rng.standard_normal((n_pages, hk, ps, d)), ct) for _ in "kv")
  cache = paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v)
  batch = paged.PagedBatch(i32([0, new]), i32([length]), i32(t), n_rows=new, max_new=new, max_len=length)
  x, outs = rng.standard_normal((new, h, d)), []
  for bad in (None, np.nan, np.inf):
    if bad is not None: x[new // 2, 0, 3] = bad
    out = put(np.zeros((new, h, d)), qt)[0]
    paged.attention(cache, batch, put(x, qt)[0], out, h, qt)
    outs.append(get(out, (new, h, d), qt))
  for got in outs[1:]:
    assert np.isnan(got[new // 2, 0]).all()
    got[new // 2, 0] = outs[0][new // 2, 0]
    assert (got == outs[0]).all()


def test_a_new_cache_on_a_stream_of_its_own():
  """The zeros of a cache that has just been allocated are there before any call on it, whatever stream that is on and whatever the device still has to do on another: they do not come over what a call
  has appended."""
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer, Stream, synchronize
  hk, d, ps = 8, 128, 16
  x, xv = put(np.arange(3 * hk * d).reshape(1, 3 * hk, d) % 61 + 1, "float16")
  q, stream, busy = put(np.zeros((1, hk, d)), "float16")[0], Stream(), DeviceBuffer(4 << 30)
  batch = paged.PagedBatch(i32([0, 1]), i32([ps]), i32([[3]]), n_rows=1, max_new=1, max_len=ps)
  kept = []                   # (freeing one waits for the device)
  for again in range(3):      # (the first time the kernel is loaded, which may wait as well)
    synchronize()
    for _ in range(20): busy.zero_()
    cache = paged.PagedCache(4, ps, hk, d)
    kept.append(cache)
    paged.append(cache, batch, x, q, hk, "float16", stream=stream)
    synchronize()
    for pool, heads in ((cache.k, xv[0, hk:2 * hk]), (cache.v, xv[0, 2 * hk:])):
      got = get(pool, (4, hk, ps, d), "float16")
      assert (got[3, :, -1] == heads).all() and np.count_nonzero(got) == hk * d, again


def test_a_capture_without_a_reserved_workspace_is_refused():
  """The capture goes on without the call, and the batch is as it was: an eager call and a reserved, captured one give the same bits."""
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import Graph, Stream
  rng = np.random.default_rng(33)
  h, hk, d, ps, length = 4, 2, 64, 16, 3000
  t, n_pages = table(rng, [length], ps)
  (k, _), (v, _), (q, _) = (put(rng.standard_normal(s), "float16") for s in ((n_pages, hk, ps, d), (n_pages, hk, ps, d), (1, h, d)))
  cache, stream = paged.PagedCache(n_pages, ps, hk, d, k=k, v=v), Stream()
  new = lambda: (paged.PagedBatch(i32([0, 1]), i32([length]), i32(t), n_rows=1, max_new=1, max_len=length), put(np.zeros((1, h, d)), "float16")[0])
  (batch, out), (other, out2) = new(), new()
  graph = Graph(stream)
  with graph:
    with pytest.raises(RuntimeError, match="reserve"): paged.attention(cache, batch, q, out, h, "float16", stream=stream)
  paged.attention(cache, batch, q, out, h, "float16", stream=stream)
  other.reserve(cache, h)
  graph = Graph(stream)
  with graph: paged.attention(cache, other, q, out2, h, "float16", stream=stream)
  for _ in range(2): graph.launch()
  stream.synchronize()
  assert (get(out, (1, h, d), "float16") == get(out2, (1, h, d), "float16")).all() and get(out, (1, h, d), "float16").any()
  assert status() == 0


def test_a_graph_whose_batch_nobody_else_holds():
  """The graph holds cache and batch: what is allocated afterwards does not land in memory that replays write."""
  need_gpu()
  import gc
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer, Graph, Stream, synchronize
  rng = np.random.default_rng(34)
  h, hk, d, ps, length = 4, 2, 64, 16, 5000
  t, n_pages = table(rng, [length], ps)
  (k, _), (v, _), (q, _) = (put(rng.standard_normal(s), "float16") for s in ((n_pages, hk, ps, d), (n_pages, hk, ps, d), (1, h, d)))
  out, stream = put(np.zeros((1, h, d)), "float16")[0], Stream()
  def captured():
    cache, batch = paged.PagedCache(n_pages, ps, hk, d, k=k, v=v), paged.PagedBatch(i32([0, 1]), i32([length]), i32(t), n_rows=1, max_new=1, max_len=length)
    batch.reserve(cache, h)
    graph = Graph(stream)
    with graph: paged.attention(cache, batch, q, out, h, "float16", stream=stream)
    return graph, batch._ws.nbytes
  graph, size = captured()
  gc.collect()
  graph.launch()
  stream.synchronize()
  want = get(out, (1, h, d), "float16")
  assert want.any()
  others = [DeviceBuffer.result((size,), np.uint8) for _ in range(100)]      # (more than the pool waits for before it hands blocks out again)
  for o in others: sevens(o)
  synchronize()
  graph.launch()
  stream.synchronize()
  assert (get(out, (1, h, d), "float16") == want).all()
  for o in others: assert (o.numpy((size,), np.uint8) == 7).all()
  assert status() == 0


def sevens(buf):
  from tinygrad_b200 import _lib
  _lib.check(_lib.load().b200q_memset(buf.ptr, 7, buf.nbytes, None))


@pytest.mark.parametrize("qt,ct", [("float16", "float16"), ("float32", "float32")])
def test_a_length_bound_next_to_31_bits(qt, ct):
  """max_len as good as none, keys in one part: the bits of a call whose bound is the length."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(35)
  h, hk, d, ps, new, length = 32, 8, 64, 16, 700, 1000
  t, n_pages = table(rng, [length], ps)
  (k, _), (v, _), (q, _) = (put(rng.standard_normal(s), c) for s, c in (((n_pages, hk, ps, d), ct), ((n_pages, hk, ps, d), ct), ((new, h, d), qt)))
  cache, outs = paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v), []
  for most in (length, (1 << 31) - 129, (1 << 31) - 128, (1 << 31) - 1):
    out = put(np.zeros((new, h, d)), qt)[0]
    paged.attention(cache, paged.PagedBatch(i32([0, new]), i32([length]), i32(t), n_rows=new, max_new=new, max_len=most), q, out, h, qt)
    outs.append(get(out, (new, h, d), qt))
  for o in outs[1:]: assert (o == outs[0]).all()
  assert outs[0].any() and status() == 0


@pytest.mark.parametrize("qt,ct,d", [("float16", "float16", 64), ("float32", "float32", 64), ("bfloat16", "bfloat16", 32)])
@pytest.mark.parametrize("off,held", [([0, 9], 4), ([0, 200], 130), ([0, 3, 150], 100), ([-5, 30], 30), ([0, 2, 40], 2)], ids=["token rows", "chunk", "second sequence", "before the first row", "no rows"])
def test_row_offsets_outside_the_arrays(qt, ct, d, off, held):
  """Sequences with rows that the arrays do not have: those they have stand at their own positions (row i of n at length - n + i, as append puts them), status 2."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(36)
  h, hk, ps, length = 4, 2, 16, [400, 300][:len(off) - 1]
  t, n_pages = table(rng, length, ps)
  (k, kv), (v, vv), (q, qv) = (put(rng.standard_normal(s), c) for s, c in (((n_pages, hk, ps, d), ct), ((n_pages, hk, ps, d), ct), ((held, h, d), qt)))
  out = put(np.full((held + 2, h, d), 3.0), qt)[0]
  cache = paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v)
  batch = paged.PagedBatch(i32(off), i32(length), i32(t), n_rows=held, max_new=max(np.diff(off)), max_len=max(length))
  status()
  paged.attention(cache, batch, q, out, h, qt)
  got = get(out, (held + 2, h, d), qt)
  assert status() == 2 and (got[held:] == 3).all()
  rows = np.zeros((off[-1] - off[0], h, d))           # the same with all of the rows
  rows[-off[0]:held - off[0]] = qv
  want, weight, reach = (x[-off[0]:held - off[0]] for x in ref.attention(rows, kv, vv, np.array(off) - off[0], length, t, ps, d ** -0.5))
  close_attention(got[:held], want, weight, reach, d, max(length), qt, qt, "the rows that there are")


def test_a_workspace_after_offsets_that_go_back():
  """Sequences that overlap until their rounds of keys pass 2^32: status 2, and the call behind it finds the workspace as the one before had left it."""
  need_gpu()
  from tinygrad_b200 import paged
  from tinygrad_b200.runtime import DeviceBuffer
  rng = np.random.default_rng(37)
  h, hk, d, ps, rows, most = 32, 8, 32, 64, 16384, 131072
  n = 129                                     # 64 of 16384 rows (2^26 rounds each), those that go back between them, one of a single row (8 x 18 rounds)
  back, ok = np.array([0, rows] * 64 + [0, 1], np.int32), np.array([0] + [1] * n, np.int32)
  lens, long = np.array([most] * (n - 1) + [18 * 64], np.int32), np.full(n, most, np.int32)
  (k, _), (v, _) = (put(rng.standard_normal((3, hk, ps, d)), "float16") for _ in "kv")
  q, out = put(rng.standard_normal((rows, h, d)), "float16")[0], put(np.zeros((rows, h, d)), "float16")[0]
  off, length = i32(ok), i32(long)
  batch = paged.PagedBatch(off, length, i32(rng.integers(0, 3, (n, most // ps))), n_rows=rows, max_new=rows, max_len=most)
  cache = paged.PagedCache(3, ps, hk, d, k=k, v=v)
  status()
  paged.attention(cache, batch, q, out, h, "float16")
  want = get(out, (1, h, d), "float16")
  assert status() == 0 and want.any()
  off.copy_from(back), length.copy_from(lens)
  paged.attention(cache, batch, q, out, h, "float16")
  assert status() == 2
  off.copy_from(ok), length.copy_from(long)
  out.copy_from(np.zeros((rows, h, d), np.float16))
  paged.attention(cache, batch, q, out, h, "float16")
  got = get(out, (rows, h, d), "float16")
  assert (got[:1] == want).all() and not got[1:].any() and status() == 0


@pytest.mark.parametrize("qt,ct,d", [("float16", "float16", 128), ("bfloat16", "bfloat16", 64), ("float32", "float16", 128), ("float32", "float32", 32)])
@pytest.mark.parametrize("seqs", [[(1, 5000), (2, 700)], [(150, 4000)], [(1, 300), (200, 900), (9, 60)]], ids=["tokens", "keys in parts", "both kernels"])
def test_attention_in_place(qt, ct, d, seqs):
  """out is q: the bits of a call whose outputs are elsewhere."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(38)
  h, hk, ps = 8, 2, 16
  new, length = [n for n, _ in seqs], [l for _, l in seqs]
  off, n = np.concatenate([[0], np.cumsum(new)]), sum(new)
  t, n_pages = table(rng, length, ps)
  (k, _), (v, _) = (put(rng.standard_normal((n_pages, hk, ps, d)), ct) for _ in "kv")
  cache = paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v)
  batch = paged.PagedBatch(i32(off), i32(length), i32(t), n_rows=n, max_new=max(new), max_len=max(length))
  q, out = put(rng.standard_normal((n, h, d)), qt)[0], put(np.zeros((n, h, d)), qt)[0]
  paged.attention(cache, batch, q, out, h, qt)
  paged.attention(cache, batch, q, q, h, qt)
  assert (get(q, (n, h, d), qt) == get(out, (n, h, d), qt)).all() and status() == 0


@pytest.mark.parametrize("qt,ct,d", [("float16", "float16", 128), ("bfloat16", "bfloat16", 64), ("float32", "float16", 128), ("float32", "float32", 64), ("float32", "bfloat16", 32)])
@pytest.mark.parametrize("seqs,bounds", [([(1, 513), (1, 70)], (1, 131072)), ([(1, 900), (3, 33), (0, 5)], (300, 5000)), ([(200, 700), (1, 300)], (4096, 131072)), ([(40, 2000)], (41, 2001)), ([(2, 2)], (2, 65536))],
                         ids=["tokens", "tokens with room for prompts", "a step's bounds", "one more", "a short one"])
def test_attention_with_bounds_above_its_tables(qt, ct, d, seqs, bounds):
  """What a captured step has: the bounds decide which kernels run and how the keys are split, the tables what they do."""
  need_gpu()
  attend(seqs, 8, 2, d, 16, qt, ct, seed=d, bounds=bounds)


@pytest.mark.parametrize("rotate_here", [True, False])
def test_norms_in_front_of_the_contiguous_cache(rotate_here):
  """head_norm_rope over the rows of b200q_attn_prefill, in place: with its rotation (prefill is told to rotate nothing: rope_dim 0) or without (prefill rotates)."""
  need_gpu()
  from tinygrad_b200 import _lib, paged
  from tinygrad_b200.runtime import DeviceBuffer
  rng = np.random.default_rng(39)
  h, hk, d, n, start, ctx = 8, 2, 128, 90, 30, 160
  width = (h + 2 * hk) * d
  rope, w = cos_sin(ctx, d), rng.uniform(0.5, 1.5, (2, d)).astype(np.float16)
  rb, wq, wk = DeviceBuffer.from_numpy(rope), DeviceBuffer.from_numpy(w[0]), DeviceBuffer.from_numpy(w[1])
  before = rng.standard_normal((2, hk, ctx, d)).astype(np.float16)
  k, v = DeviceBuffer.from_numpy(before[0]), DeviceBuffer.from_numpy(before[1])
  x, xv = put(rng.standard_normal((n, h + 2 * hk, d)), "float32")
  q, out = DeviceBuffer.empty((n, h * d), np.float32), DeviceBuffer.empty((n, h * d), np.float32)
  paged.head_norm_rope(x, x, n, h, hk, d, q_norm=wq, k_norm=wk, norm_eps=1e-6, rope=rb if rotate_here else None, positions=i32(start + np.arange(n)) if rotate_here else None, x_stride=width, out_stride=width)
  _lib.check(_lib.load().b200q_attn_prefill(x.ptr, k.ptr, v.ptr, _lib.F16, rb.ptr, start, n, h, hk, d, 0 if rotate_here else d, ctx, q.ptr, out.ptr, _lib.F32, None))
  rot, now = rope[start:start + n], x.numpy((n, h + 2 * hk, d), np.float32).astype(np.float64)
  assert (now[:, h + hk:] == xv[:, h + hk:]).all()
  for a, b, ww in ((0, h, w[0]), (h, h + hk, w[1])):
    here = rot if rotate_here else None
    close_rows(now[:, a:b], ref.rotate(ref.head_norm(xv[:, a:b], ww, 1e-6), here), reach_of(xv[:, a:b], ww, 1e-6, here), "float32", "rows")
  kc, vc = k.numpy().astype(np.float64), v.numpy().astype(np.float64)
  new = slice(start, start + n)
  assert (kc[:, :start] == before[0][:, :start]).all() and (vc[:, new] == xv[:, h + hk:].astype(np.float16).transpose(1, 0, 2)).all()
  kw = ref.rotate(ref.head_norm(xv[:, h:h + hk], w[1], 1e-6), rot)
  close_rows(kc[:, new].transpose(1, 0, 2), kw, reach_of(xv[:, h:h + hk], w[1], 1e-6, rot), "float16", "keys")
  # queries as prefill takes them: those of the rows, or (its own rotation, 32 bits) within 2^-22 of (|a| + |b|) of them -- 64-bit values here, a score's walk covers that
  qs = now[:, :h] if rotate_here else ref.rotate(now[:, :h], rot)
  want, weight, reach = ref.attention(qs, kc[None], vc[None], [0, n], [start + n], np.zeros((1, 1), int), ctx, d ** -0.5)
  close_attention(out.numpy((n, h, d), np.float32).astype(np.float64), want, weight, reach, d, start + n, "float32", "float32", "attention")


@pytest.mark.parametrize("qt,ct,d", [("float16", "float16", 32), ("float16", "float16", 128), ("float32", "float32", 64)])
@pytest.mark.parametrize("new", [[1, 2], [150, 3]])
def test_offsets_of_sequences_that_are_not_there(qt, ct, d, new):
  """A table of more sequences than there are, whose last entries are 0: the offsets go back (status 2), nothing overlaps, and the rows get their answers."""
  need_gpu()
  from tinygrad_b200 import paged
  rng = np.random.default_rng(40)
  h, hk, ps, length, n = 4, 2, 16, [300, 2500], sum(new)
  t, n_pages = table(rng, length, ps)
  (k, kv), (v, vv), (q, qv) = (put(rng.standard_normal(s), c) for s, c in (((n_pages, hk, ps, d), ct), ((n_pages, hk, ps, d), ct), ((n, h, d), qt)))
  out = put(np.zeros((n, h, d)), qt)[0]
  batch = paged.PagedBatch(i32([0, new[0], n] + [0] * 40), i32(length + [0] * 40), i32(np.concatenate([t, np.zeros((40, t.shape[1]), int)])), n_rows=n, max_new=max(new), max_len=max(length))
  status()
  paged.attention(paged.PagedCache(n_pages, ps, hk, d, ct, k=k, v=v), batch, q, out, h, qt)
  want, weight, reach = ref.attention(qv, kv, vv, [0, new[0], n], length, t, ps, d ** -0.5)
  close_attention(get(out, (n, h, d), qt), want, weight, reach, d, max(length), qt, qt, "rows")
  assert status() == 2
