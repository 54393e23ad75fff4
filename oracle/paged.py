"""The paged-cache operators in numpy, 64 bits: norms of heads, half-split rotation, appending to pages, attention of a ragged batch over pages."""
import numpy as np


def bf16_values(bits: np.ndarray) -> np.ndarray:
  return (np.asarray(bits).astype(np.uint32) << 16).view(np.float32)


def bf16_bits(x: np.ndarray) -> np.ndarray:
  """Round to nearest, ties to even; NaN stays NaN."""
  x = np.asarray(x, dtype=np.float32)
  u = x.view(np.uint32)
  r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
  return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def head_norm(x, w, eps):
  """x [..., dim]: RMSNorm over the last axis (tinygrad/nn/__init__.py:300-304); w None: x."""
  x = np.asarray(x, dtype=np.float64)
  return x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, dtype=np.float64)


def rotate(x, cos_sin):
  """x [n, heads, dim], cos_sin [n, r]: half-split pairs in the first r values (tinygrad/llm/model.py:29-33)."""
  if cos_sin is None: return x
  r = cos_sin.shape[-1] // 2
  c, s = (np.asarray(cos_sin, dtype=np.float64)[:, None, i:i + r] for i in (0, r))
  a, b = x[..., :r], x[..., r:2 * r]
  return np.concatenate([a * c - b * s, b * c + a * s, x[..., 2 * r:]], axis=-1)


def rows_of(row_off, length):
  """(sequence, position) of every row of the batch, in order."""
  return [(s, int(length[s]) - (int(row_off[s + 1]) - int(row_off[s])) + i) for s in range(len(length)) for i in range(int(row_off[s + 1]) - int(row_off[s]))]


def gather(pool, pages, n, page_size):
  """pool [page][head][slot][dim] -> [head][n][dim] of a sequence's first n positions; pages that do not exist read as zeros."""
  out = np.zeros((pool.shape[1], n, pool.shape[3]))
  for j in range(n):
    p = pages[j // page_size]
    if 0 <= p < pool.shape[0]: out[:, j] = pool[p, :, j % page_size]
  return out


def attention(q, k_pool, v_pool, row_off, length, pages, page_size, scale):
  """q [rows][heads][dim] -> (out, sum_j p_j |v_j| (what errors of p are relative to), largest sum_d |q_d k_d| scale of a row's keys)."""
  n, heads, dim = q.shape
  group = heads // k_pool.shape[1]
  out, weight, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, heads))
  cache = {}
  for row, (s, pos) in enumerate(rows_of(row_off, length)):
    if pos < 0: continue
    if s not in cache: cache = {s: [gather(p, pages[s], int(length[s]), page_size) for p in (k_pool, v_pool)]}
    k, v = (x[:, :pos + 1] for x in cache[s])
    for h in range(heads):
      kk, vv = k[h // group], v[h // group]
      w = kk @ q[row, h].astype(np.float64) * scale
      e = np.exp(w - w.max())
      e /= e.sum()
      out[row, h], weight[row, h], reach[row, h] = e @ vv, e @ np.abs(vv), (np.abs(kk) @ np.abs(q[row, h].astype(np.float64))).max() * scale
  return out, weight, reach
