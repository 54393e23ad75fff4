"""A paged KV cache and what reads and writes it: for serving sequences of different lengths in one batch.

`PagedCache` holds one block's keys and values in pages of `page_size` positions, `PagedBatch` the tables that say which rows (new tokens) and pages belong to
which sequence; all of it lives on the device, so that a captured step follows the lengths.  `append` takes the projections of the new tokens into the pages (norms of the heads and
rotation on the way), `attention` is the attention of the new tokens over the pages -- TransformerBlock._attention of tinygrad/llm/model.py:167-207 for a
ragged batch --, `head_norm_rope` the norms and the rotation alone, for caches that are not paged.

Buffers are DeviceBuffers or foreign tensors of the current device, held to the type that the call names where they say theirs (bf16 values are uint16 in a DeviceBuffer), or raw addresses
(`runtime.ptr_of`; the tables of a batch and `rope` are asked for their shapes and cannot be).  Calls launch on `stream` and return at
once; a batch's workspace serves one call at a time: streams and graphs that may run together need a PagedBatch each.  A captured call's cache and batch live as long as the graph:
`runtime.Graph` keeps them; under another kind of capture the caller does.  Rows, outputs and angles are the caller's to keep, as with any call."""
import ctypes, struct
import numpy as np
from . import _lib
from ._lib import check, F32, F16, BF16
from .runtime import DeviceBuffer, Graph, ptr_of, stream_ptr, synchronize

DTYPES = {"float32": F32, "float16": F16, "bfloat16": BF16}
_NP = {F32: np.float32, F16: np.float16, BF16: np.uint16}
_SIZE = {F32: 4, F16: 2, BF16: 2}
_TYPE = {**DTYPES, **{t: t for t in _SIZE}}
# The calls of a decode step are as long as what Python does for them: types are looked up, not taken apart, the library's entries are bound once, and their arguments are packed into bytes
# (0.15 us; a ctypes structure takes 0.7).
_entry = {}
_LETTERS = {ctypes.c_void_p: "P", ctypes.c_int: "i", ctypes.c_int64: "q", ctypes.c_float: "f", ctypes.c_size_t: "N"}


def _packer(args):
  p = struct.Struct("@" + "".join(_LETTERS[t] for _, t in args._fields_))
  assert p.size == ctypes.sizeof(args), args
  return p.pack


_append_args, _norm_args, _attn_args = (_packer(a) for a in (_lib.PagedAppendArgs, _lib.HeadNormArgs, _lib.PagedAttnArgs))
WORKSPACE_HEAD = 16384      # bytes of b200q_paged_attention's workspace that begin as zeros


def _fn(name: str):
  """The library's entry `name`, which takes its arguments' structure as bytes."""
  f = _entry.get(name)
  if f is None:
    kinds = [ctypes.c_char_p if a in (ctypes.POINTER(_lib.PagedAppendArgs), ctypes.POINTER(_lib.HeadNormArgs), ctypes.POINTER(_lib.PagedAttnArgs)) else a for a in _lib.SIGNATURES[name][1]]
    f = _entry[name] = ctypes.CFUNCTYPE(_lib.SIGNATURES[name][0], *kinds)((name, _lib.load()))
  return f


def _dtype(d) -> int:
  t = _TYPE.get(d)
  if t is None: raise ValueError(f"unknown element type {d!r}: float32, float16 or bfloat16")
  return t


def _ptr(o) -> int:
  if type(o) is DeviceBuffer: return o.ptr
  try:
    if not o.is_cuda and not o.is_pinned(): raise ValueError("a tensor on the host: the kernels read and write device memory, or host memory that is page-locked")
    return o.data_ptr()
  except AttributeError: return ptr_of(o)


def _short(o, nbytes: int, what: str) -> None:
  have = getattr(o, "nbytes", None)      # (a raw address says nothing)
  if type(have) is int and have < nbytes:
    if hasattr(o, "untyped_storage"): have = o.untyped_storage().nbytes() - o.storage_offset() * o.element_size()      # a view of rows that lie apart: nbytes counts its values alone
    if have < nbytes: raise ValueError(f"{what} has {have} bytes, needs {nbytes}")


_INT32 = -1
_NAMES = {F32: ("float32", "float"), F16: ("float16", "half"), BF16: ("bfloat16", "uint16"), _INT32: ("int32", "int")}
_same = {t: set() for t in _NAMES}       # by element type: what objects of it have said that their elements are


def _typed(o, t: int, what: str) -> None:
  d = getattr(o, "dtype", None)          # (a raw address says nothing, bytes are anything)
  if d is None or d in _same[t]: return
  name = str(d).rsplit(".", 1)[-1]
  if name not in _NAMES[t] and name != "uint8": raise TypeError(f"{what} has elements of {d}, and the call says {_NAMES[t][0]}")
  if name != "uint8": _same[t].add(d)


def _dense(o, what: str) -> None:
  f = getattr(o, "is_contiguous", None)
  if f is not None and not f(): raise ValueError(f"{what} is not contiguous")


def _rows(o, t: int, nbytes: int, stride: int, what: str) -> int:
  """The address of an array of type t that the call reads or writes nbytes of.  stride 0: its values lie back to back."""
  try:      # a tensor that is as it should be: all of it in a quarter of a microsecond
    if o.dtype in _same[t] and o.is_cuda and (stride or o.is_contiguous()) and o.nbytes >= nbytes: return o.data_ptr()
  except AttributeError: pass
  _typed(o, t, what)
  if not stride: _dense(o, f"{what}, whose stride is not given,")
  _short(o, nbytes, what)
  return _ptr(o)


def _angles(rope) -> tuple:
  """(address, rotated dimensions, positions) of a table cos || sin."""
  if rope is None: return 0, 0, 0
  try: n, dim = rope.shape
  except (AttributeError, ValueError): raise ValueError(f"rope is a table [positions, rotated dimensions], got {getattr(rope, 'shape', rope)!r}") from None
  return _rows(rope, F32, 4 * n * dim, 0, "rope"), dim, n


def _kept(stream, *objects) -> None:
  """A graph that is being captured on the stream keeps the objects."""
  graph = Graph.open.get(stream_ptr(stream))
  if graph is not None: graph.kept += objects


def _fits(*values) -> None:
  if max(values) >= 1 << 31: raise ValueError(f"{max(values)} does not fit into 31 bits")


_words = set()     # types that have been seen to be int32


def _int32(o, what: str):
  t = getattr(o, "dtype", None)
  if t is not None and t not in _words:
    if not str(t).endswith("int32") or str(t).endswith("uint32"): raise TypeError(f"{what} is a table of int32, got {t}")
    _words.add(t)
  return o


class PagedCache:
  """One block's keys and values: pools `k` and `v` of n_pages pages (allocated here, zeroed, unless given).  strides: elements from page to page, KV head to KV head and slot to
  slot; the default is [page][head][slot][head_dim]."""
  def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype="float16", k=None, v=None, strides: tuple = None):
    if min(n_pages, page_size, n_kv_heads, head_dim) <= 0: raise ValueError("pages, page size, heads and head size are at least 1")
    _fits(n_pages, page_size, n_kv_heads, head_dim)
    if (k is None) != (v is None): raise ValueError("give both pools or neither")
    self.n_pages, self.page_size, self.n_kv_heads, self.head_dim, self.dtype = n_pages, page_size, n_kv_heads, head_dim, _dtype(dtype)
    page, head, row = self.strides = tuple(strides) if strides is not None else (n_kv_heads * page_size * head_dim, page_size * head_dim, head_dim)
    if min(self.strides) < head_dim: raise ValueError(f"strides {self.strides} are shorter than a head")
    last = (n_pages - 1) * page + (n_kv_heads - 1) * head + (page_size - 1) * row + head_dim
    if k is None:
      k, v = (DeviceBuffer.empty((last,), _NP[self.dtype], zero=True) for _ in range(2))
      synchronize()                      # whatever stream the first call is on: zeros that come late would go over what it has appended
    self.k, self.v = k, v
    at = [_rows(x, self.dtype, last * _SIZE[self.dtype], strides is not None, what) for x, what in ((k, "k"), (v, "v"))]
    self.desc = _lib.PagedCacheDesc(*at, self.dtype, n_pages, page_size, n_kv_heads, head_dim, page, head, row)
    self.ref, self._key = ctypes.byref(self.desc), (self.dtype, page_size, n_kv_heads, head_dim)


class PagedBatch:
  """Which rows and pages belong to which sequence.  row_off int32 [n_seqs + 1]: sequence s has the rows row_off[s] .. row_off[s + 1] - 1, its new tokens; length int32 [n_seqs]: its
  tokens in all, the new ones among them; pages int32 [n_seqs, most pages of a sequence].  The tables are read when the work runs and may change between calls (or replays of a
  graph); n_rows (rows of the row arrays), max_new and max_len (of any sequence) are bounds that hold for all of them."""
  def __init__(self, row_off, length, pages, n_rows: int, max_new: int, max_len: int):
    if min(n_rows, max_new, max_len) < 0: raise ValueError("bounds are not negative")
    _fits(n_rows, max_new, max_len)
    (n_seqs,), (seqs, table) = length.shape, pages.shape
    if seqs != n_seqs or tuple(row_off.shape) != (n_seqs + 1,): raise ValueError(f"row_off {tuple(row_off.shape)}, length {tuple(length.shape)} and pages {tuple(pages.shape)} do not match")
    if n_seqs and table < 1: raise ValueError("a sequence has at least one entry in the table of pages")
    for x, what in ((row_off, "row_off"), (length, "length"), (pages, "pages")): _dense(x, what)
    self.row_off, self.length, self.pages = _int32(row_off, "row_off"), _int32(length, "length"), _int32(pages, "pages")
    self.n_seqs, self.n_rows, self.max_new, self.max_len = n_seqs, n_rows, max_new, max_len
    self.desc = _lib.PagedBatchDesc(_ptr(row_off), _ptr(length), _ptr(pages), n_seqs, table, n_rows, max_new, max_len)
    self.ref = ctypes.byref(self.desc)
    self._ws, self._ready, self._old = None, set(), []

  def reserve(self, cache: PagedCache, n_heads: int, q_dtype="float32") -> None:
    """Allocates the workspace that `attention` needs for such a cache and such rows, of whatever type.  A call's first time does so otherwise; one that is captured cannot."""
    _dtype(q_dtype)
    if self._reserve(cache, n_heads, None): synchronize()        # whatever stream the first call is on

  def _reserve(self, cache: PagedCache, n_heads: int, stream) -> bool:
    """True: a new workspace, whose zeros are on their way on `stream`."""
    need = _fn("b200q_paged_attention_workspace_bytes")(cache.ref, self.ref, n_heads)
    fresh = need > 0 and (self._ws is None or self._ws.nbytes < need)
    if fresh:
      lib, capturing = _lib.load(), ctypes.c_int()
      if stream is not None: check(lib.b200q_stream_is_capturing(stream_ptr(stream), ctypes.byref(capturing)))
      if capturing.value: raise RuntimeError("a captured call allocates nothing: PagedBatch.reserve goes before the capture")
      ws = DeviceBuffer.result((need,), np.uint8, stream)      # (from the pool: a batch may live as briefly as a step)
      check(lib.b200q_memset(ws.ptr, 0, WORKSPACE_HEAD, stream_ptr(stream)))
      if self._ws is not None: self._old.append(self._ws)      # graphs may hold it
      self._ws = ws
    self._ready.add((cache._key, n_heads))
    return fresh


def append(cache: PagedCache, batch: PagedBatch, x, q, n_heads: int, x_dtype="float32", q_dtype=None, rope=None, q_norm=None, k_norm=None, norm_eps: float = 0.0, x_stride: int = 0,
           q_stride: int = 0, flags: int = 0, stream=None) -> None:
  """x rows [q | k | v] (x_dtype, x_stride elements apart, 0: back to back) of the batch's new tokens: q rows normed and rotated to `q` (q_dtype, the same as x's unless given), k likewise and v to
  the pages.  rope: fp32 [positions, rotated dimensions], cos || sin (`model.precompute_freqs_cis`), or None; q_norm / k_norm: fp16 [head_dim], the weights of an RMSNorm over each head, or None."""
  xt = _dtype(x_dtype)
  qt = xt if q_dtype is None else _dtype(q_dtype)
  n, d = batch.n_rows, cache.head_dim
  row, q_row = (n_heads + 2 * cache.n_kv_heads) * d, n_heads * d
  xp = _rows(x, xt, ((n - 1) * (x_stride or row) + row) * _SIZE[xt] if n else 0, x_stride, "x")
  qp = _rows(q, qt, ((n - 1) * (q_stride or q_row) + q_row) * _SIZE[qt] if n else 0, q_stride, "q")
  a = _append_args(xp, qp, xt, qt, x_stride, q_stride, n_heads, norm_eps, 0 if q_norm is None else _norm(q_norm, d), 0 if k_norm is None else _norm(k_norm, d), *_angles(rope))
  if Graph.open: _kept(stream, cache, batch)
  rc = _fn("b200q_paged_append")(cache.ref, batch.ref, a, flags, 0 if stream is None else stream_ptr(stream))
  if rc: check(rc)


def attention(cache: PagedCache, batch: PagedBatch, q, out, n_heads: int, q_dtype="float32", out_dtype=None, scale: float = 0.0, q_stride: int = 0, out_stride: int = 0, flags: int = 0,
              stream=None) -> None:
  """out[row][head] = softmax(scale q . k) v over the positions up to the row's own (scale 0: head_dim ** -0.5); out_dtype is q's unless given, out may be q.  16-bit queries, pages and outputs: a probability
  is rounded to the pages' type; out_dtype "float32" keeps 32 bits throughout."""
  qt = _dtype(q_dtype)
  ot = qt if out_dtype is None else _dtype(out_dtype)
  n, row = batch.n_rows, n_heads * cache.head_dim
  qp = _rows(q, qt, ((n - 1) * (q_stride or row) + row) * _SIZE[qt] if n else 0, q_stride, "q")
  op = _rows(out, ot, ((n - 1) * (out_stride or row) + row) * _SIZE[ot] if n else 0, out_stride, "out")
  if (cache._key, n_heads) not in batch._ready: batch._reserve(cache, n_heads, stream)
  ws = batch._ws
  a = _attn_args(qp, op, qt, ot, q_stride, out_stride, n_heads, scale, *((0, 0) if ws is None else (ws.ptr, ws.nbytes)))
  if Graph.open: _kept(stream, cache, batch)
  rc = _fn("b200q_paged_attention")(cache.ref, batch.ref, a, flags, 0 if stream is None else stream_ptr(stream))
  if rc: check(rc)


def _norm(w, d: int) -> int:
  return _rows(w, F16, 2 * d, 0, "a float16 norm weight")


def head_norm_rope(x, out, n_rows: int, n_heads: int, n_kv_heads: int, head_dim: int, x_dtype="float32", out_dtype=None, q_norm=None, k_norm=None, norm_eps: float = 0.0, rope=None,
                   positions=None, x_stride: int = 0, out_stride: int = 0, flags: int = 0, stream=None) -> None:
  """The norms and the rotation of the first n_heads (queries) + n_kv_heads (keys) heads of every row, from x to out, which may be x (strides and types as they are, then).  positions: int32
  [n_rows] with rope."""
  xt = _dtype(x_dtype)
  ot = xt if out_dtype is None else _dtype(out_dtype)
  row = (n_heads + n_kv_heads) * head_dim
  xp = _rows(x, xt, ((n_rows - 1) * (x_stride or row) + row) * _SIZE[xt] if n_rows > 0 else 0, x_stride, "x")
  op = _rows(out, ot, ((n_rows - 1) * (out_stride or row) + row) * _SIZE[ot] if n_rows > 0 else 0, out_stride, "out")
  angles, rope_dim, rope_len = _angles(rope)
  a = _norm_args(xp, op, xt, ot, x_stride, out_stride, n_rows, n_heads, n_kv_heads, head_dim, norm_eps, 0 if q_norm is None else _norm(q_norm, head_dim),
                 0 if k_norm is None else _norm(k_norm, head_dim), angles, rope_dim, rope_len, 0 if positions is None else _rows(positions, _INT32, 4 * max(n_rows, 0), 0, "positions"))
  rc = _fn("b200q_head_norm_rope")(a, flags, 0 if stream is None else stream_ptr(stream))
  if rc: check(rc)
