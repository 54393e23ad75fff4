"""What the paged-cache entry points refuse, without a device, and the host side of their classes."""
import ctypes
import numpy as np
import pytest
from tinygrad_b200 import _lib, build, paged
from tinygrad_b200._lib import F32, F16, BF16


@pytest.fixture(scope="module")
def lib():
  build.build_lib()
  return _lib.load()


P = 0x1000


def cache(**kw):
  c = _lib.PagedCacheDesc(P, P, F16, 10, 16, 2, 64, 2 * 16 * 64, 16 * 64, 64)
  for k, v in kw.items(): setattr(c, k, v)
  return c


def batch(**kw):
  b = _lib.PagedBatchDesc(P, P, P, 2, 4, 3, 2, 60)
  for k, v in kw.items(): setattr(b, k, v)
  return b


def call(fn, *structs): return fn(*[None if s is None else ctypes.byref(s) for s in structs], 0, None)


BAD_CACHE = [(dict(k=None), -1), (dict(v=None), -1), (dict(dtype=3), -1), (dict(n_pages=0), -1), (dict(page_size=0), -1), (dict(n_kv_heads=-1), -1), (dict(head_dim=96), -2), (dict(head_dim=0), -2),
             (dict(row_stride=32), -2), (dict(head_stride=0), -2), (dict(page_stride=-2048), -2), (dict(row_stride=68), -3), (dict(k=P + 8), -3)]
BAD_BATCH = [(dict(row_off=None), -1), (dict(length=None), -1), (dict(pages=None), -1), (dict(n_seqs=-1), -1), (dict(n_rows=-1), -1), (dict(table_stride=0), -1), (dict(max_new=0), -1), (dict(max_len=-1), -1),
             (dict(length=P + 2), -3)]


@pytest.mark.parametrize("change,code", [(("cache", c), e) for c, e in BAD_CACHE] + [(("batch", c), e) for c, e in BAD_BATCH])
def test_caches_and_batches_that_are_refused(lib, change, code):
  c, b = cache(**change[1] if change[0] == "cache" else {}), batch(**change[1] if change[0] == "batch" else {})
  assert call(lib.b200q_paged_append, c, b, _lib.PagedAppendArgs(P, P, F32, F32, 0, 0, 4)) == code
  assert call(lib.b200q_paged_attention, c, b, _lib.PagedAttnArgs(P, P, F32, F32, 0, 0, 4, 0.0, P, 1 << 30)) == code
  assert lib.b200q_paged_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 4) == 0


@pytest.mark.parametrize("change,code", [(dict(x=None), -1), (dict(q=None), -1), (dict(x_dtype=5), -1), (dict(q_dtype=-1), -1), (dict(n_heads=0), -1), (dict(x_stride=8 * 64 - 1), -2), (dict(q_stride=255), -2),
                                         (dict(rope=P, rope_dim=0, rope_len=8), -1), (dict(rope=P, rope_dim=32, rope_len=0), -1), (dict(rope=P, rope_dim=31, rope_len=8), -2), (dict(rope=P, rope_dim=66, rope_len=8), -2),
                                         (dict(rope=P + 1, rope_dim=32, rope_len=8), -3), (dict(x=P + 2), -3), (dict(q=P + 3), -3), (dict(k_norm=P + 1), -3), (dict(q=2 * P, q_stride=512), -1),
                                         (dict(q=2 * P, q_dtype=F16, x_stride=512, q_stride=512), -1), (dict(n_heads=1 << 28), -2)])
def test_append_refuses(lib, change, code):
  a = _lib.PagedAppendArgs(2 * P, P, F32, F32, 0, 0, 4)
  for k, v in change.items(): setattr(a, k, v)
  if change.get("q") == 2 * P and "x_stride" not in change: a.x_stride = 600      # in place with other strides
  assert call(lib.b200q_paged_append, cache(), batch(), a) == code


@pytest.mark.parametrize("change,code", [(dict(q=None), -1), (dict(out=None), -1), (dict(q_dtype=9), -1), (dict(out_dtype=9), -1), (dict(n_heads=3), -1), (dict(n_heads=0), -1), (dict(scale=-1.0), -1),
                                         (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(q_stride=255), -2), (dict(out_stride=10), -2), (dict(q=P + 2), -3), (dict(out=P + 1), -3),
                                         (dict(workspace=P + 16), -3), (dict(workspace=None), -6), (dict(workspace_bytes=100), -6)])
def test_attention_refuses(lib, change, code):
  a = _lib.PagedAttnArgs(P, P, F32, F32, 0, 0, 4, 0.0, P, 1 << 30)
  for k, v in change.items(): setattr(a, k, v)
  b = batch(max_len=100000, table_stride=7000)      # long enough to be split over CTAs
  assert lib.b200q_paged_attention_workspace_bytes(ctypes.byref(cache()), ctypes.byref(b), 4) > 100
  assert call(lib.b200q_paged_attention, cache(), b, a) == code


@pytest.mark.parametrize("change,code", [(dict(x=None), -1), (dict(out=None), -1), (dict(n_rows=-1), -1), (dict(n_heads=-1), -1), (dict(n_heads=0, n_kv_heads=0), -1), (dict(x_dtype=7), -1), (dict(out_dtype=7), -1),
                                         (dict(head_dim=48), -2), (dict(x_stride=100), -2), (dict(out_stride=100), -2), (dict(rope=P, rope_dim=64, rope_len=9), -1), (dict(rope=P, rope_dim=65, rope_len=9, positions=P), -2),
                                         (dict(rope=P, rope_dim=64, rope_len=9, positions=P + 1), -3), (dict(x=P + 1), -3), (dict(q_norm=P + 1), -3), (dict(out=2 * P, out_stride=1000), -1),
                                         (dict(out=2 * P, out_dtype=F16), -1)])
def test_head_norm_rope_refuses(lib, change, code):
  a = _lib.HeadNormArgs(2 * P, P, F32, F32, 0, 0, 5, 4, 2, 64)
  for k, v in change.items(): setattr(a, k, v)
  assert lib.b200q_head_norm_rope(ctypes.byref(a), 0, None) == code


@pytest.mark.parametrize("kv_dtype", [F16, F32])
@pytest.mark.parametrize("n_heads,change", [(64, dict(n_seqs=(1 << 31) - 1, n_rows=(1 << 31) - 1, max_new=1)),
                                            (2, dict(n_seqs=(1 << 31) - 1, n_rows=(1 << 31) - 1, max_new=100, max_len=(1 << 31) - 1))])
def test_work_past_31_bits_is_refused(lib, kv_dtype, n_heads, change):
  """Tiles and rounds that no launch can have: an error, not a count that wrapped around (to 0: a division by it)."""
  c, b = cache(dtype=kv_dtype), batch(**change)
  lib.b200q_paged_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), n_heads)
  assert call(lib.b200q_paged_attention, c, b, _lib.PagedAttnArgs(P, P, F32, F32, 0, 0, n_heads, 0.0, P, (1 << 63) - 1)) == -6


def test_nothing_to_do_is_fine(lib):
  for b in (batch(n_seqs=0, row_off=None, length=None, pages=None), batch(n_rows=0)):
    assert call(lib.b200q_paged_append, cache(), b, _lib.PagedAppendArgs(None, None, F32, F32, 0, 0, 4)) == 0
    assert call(lib.b200q_paged_attention, cache(), b, _lib.PagedAttnArgs(None, None, F32, F32, 0, 0, 4)) == 0
  assert lib.b200q_head_norm_rope(ctypes.byref(_lib.HeadNormArgs(None, None, F32, F32, 0, 0, 0, 4, 2, 64)), 0, None) == 0


def test_structs_have_the_header_s_layout(tmp_path):
  import pathlib, shutil, subprocess
  cc = shutil.which("gcc") or shutil.which("cc")
  if not cc: pytest.skip("no host C compiler")
  hdr = pathlib.Path(__file__).resolve().parent.parent / "include" / "b200q.h"
  structs = {"b200q_paged_cache": _lib.PagedCacheDesc, "b200q_paged_batch": _lib.PagedBatchDesc, "b200q_paged_append_args": _lib.PagedAppendArgs, "b200q_head_norm_args": _lib.HeadNormArgs,
             "b200q_paged_attn_args": _lib.PagedAttnArgs}
  lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{hdr}"', "int main(void) {"]
  for c, t in structs.items():
    lines += [f'printf("{c} %zu\\n", sizeof({c}));'] + [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in t._fields_]
  (tmp_path / "l.c").write_text("\n".join(lines + ["return 0;", "}"]))
  subprocess.run([cc, "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
  got = dict(l.split() for l in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines())
  for c, t in structs.items():
    assert int(got[c]) == ctypes.sizeof(t), c
    for f, _ in t._fields_: assert int(got[f"{c}.{f}"]) == getattr(t, f).offset, f"{c}.{f}"


class Fake:
  """A buffer that is only asked for its address, size and type."""
  def __init__(self, shape, dtype): self.shape, self.dtype, self.ptr, self.nbytes = tuple(shape), np.dtype(dtype), P, int(np.prod(shape)) * np.dtype(dtype).itemsize


def test_python_side_refuses(lib):
  i = lambda *s: Fake(s, np.int32)
  with pytest.raises(ValueError, match="both pools"): paged.PagedCache(4, 16, 2, 64, k=Fake((4, 2, 16, 64), np.float16))
  with pytest.raises(ValueError, match="element type"): paged.PagedCache(4, 16, 2, 64, "int8", k=P, v=P)
  with pytest.raises(ValueError, match="at least 1"): paged.PagedCache(4, 0, 2, 64, k=P, v=P)
  with pytest.raises(ValueError, match="k has"): paged.PagedCache(4, 16, 2, 64, k=Fake((4, 2, 16, 63), np.float16), v=P)
  with pytest.raises(ValueError, match="shorter"): paged.PagedCache(4, 16, 2, 64, k=P, v=P, strides=(2048, 1024, 32))
  with pytest.raises(ValueError, match="do not match"): paged.PagedBatch(i(2), i(2), i(2, 5), 2, 1, 9)
  with pytest.raises(ValueError, match="do not match"): paged.PagedBatch(i(3), i(2), i(3, 5), 2, 1, 9)
  with pytest.raises(ValueError, match="at least one"): paged.PagedBatch(i(3), i(2), i(2, 0), 2, 1, 9)
  with pytest.raises(ValueError, match="bounds"): paged.PagedBatch(i(3), i(2), i(2, 5), 2, -1, 9)
  with pytest.raises(TypeError, match="int32"): paged.PagedBatch(i(3), Fake((2,), np.int64), i(2, 5), 2, 1, 9)
  c, b = paged.PagedCache(4, 16, 2, 64, k=P, v=P), paged.PagedBatch(i(3), i(2), i(2, 5), 2, 1, 9)
  with pytest.raises(ValueError, match="x has"): paged.append(c, b, Fake((2, 7, 64), np.float32), P, 4)
  with pytest.raises(ValueError, match="q has"): paged.append(c, b, P, Fake((1, 4, 64), np.float32), 4)
  with pytest.raises(TypeError, match="float16"): paged.append(c, b, P, P, 4, q_norm=Fake((64,), np.float32))
  with pytest.raises(ValueError, match="out has"): paged.attention(c, b, P, Fake((2, 4, 63), np.float32), 4)
  with pytest.raises(ValueError, match="positions has"): paged.head_norm_rope(P, P, 5, 4, 2, 64, rope=Fake((9, 64), np.float32), positions=i(4))
  with pytest.raises(_lib.B200QError): paged.attention(c, b, P, P, 3)
  for big in ((1 << 31, 1, 9), (2, 1 << 32, 9), (2, 1, (1 << 32) + 9)):
    with pytest.raises(ValueError, match="31 bits"): paged.PagedBatch(i(3), i(2), i(2, 5), *big)
  with pytest.raises(ValueError, match="31 bits"): paged.PagedCache((1 << 32) + 4, 16, 2, 64, k=P, v=P)


def test_views_of_rows_that_lie_apart():
  """A foreign tensor's nbytes counts its values, not what lies between its rows."""
  import torch
  big = torch.zeros(3, 100)
  paged._short(big[:, :64], (2 * 100 + 64) * 4, "x")
  paged._short(big[:, 36:], (2 * 100 + 64) * 4, "x")
  with pytest.raises(ValueError, match="x has"): paged._short(big[:, 37:], (2 * 100 + 64) * 4, "x")
  with pytest.raises(ValueError, match="x has"): paged._short(big[1:, :64], (2 * 100 + 64) * 4, "x")


def test_tables_of_angles_that_are_refused(lib):
  """The rotation's table is fp32, two-dimensional and dense: anything else would be read past its end, or as other angles."""
  import torch
  c, b = paged.PagedCache(4, 16, 2, 64, k=P, v=P), paged.PagedBatch(*(Fake(s, np.int32) for s in ((3,), (2,), (2, 5))), 2, 1, 9)
  for rope, err, match in ((Fake((9, 64), np.float16), TypeError, "rope"), (Fake((9, 64), np.float64), TypeError, "rope"), (Fake((9, 64), np.uint16), TypeError, "rope"), (Fake((9 * 64,), np.float32), ValueError, "rope"),
                           (Fake((9, 2, 32), np.float32), ValueError, "rope"), (P, ValueError, "rope"), (torch.zeros(9, 128)[:, :64], ValueError, "rope"), (torch.zeros(64, 9).t(), ValueError, "rope"),
                           (torch.zeros(9, 64, dtype=torch.bfloat16), TypeError, "rope"), (torch.zeros(9, 64), ValueError, "host")):
    with pytest.raises(err, match=match): paged.append(c, b, P, P, 4, rope=rope)
    with pytest.raises(err, match=match): paged.head_norm_rope(P, P, 5, 4, 2, 64, rope=rope, positions=P)
  short = Fake((9, 64), np.float32)
  short.nbytes -= 4
  with pytest.raises(ValueError, match="rope has"): paged.append(c, b, P, P, 4, rope=short)


def test_buffers_of_other_types_than_named(lib):
  """An object that says what its elements are is held to the type argument; uint16 stands for bf16, bytes and raw addresses for anything."""
  c, b = paged.PagedCache(4, 16, 2, 64, k=P, v=P), paged.PagedBatch(*(Fake(s, np.int32) for s in ((3,), (2,), (2, 5))), 2, 1, 9)
  pool, rows = lambda t: Fake((4, 2, 16, 64), t), lambda t: Fake((2, 8, 64), t)
  for named, given in (("float16", np.uint16), ("float16", np.float32), ("bfloat16", np.float16), ("float32", np.float64), ("float32", np.int32)):
    with pytest.raises(TypeError, match="k has"): paged.PagedCache(4, 16, 2, 64, named, k=Fake((8, 2, 16, 64), given), v=P)
    with pytest.raises(TypeError, match="v has"): paged.PagedCache(4, 16, 2, 64, named, k=P, v=Fake((8, 2, 16, 64), given))
    wide = Fake((8, 8, 64), given)
    with pytest.raises(TypeError, match="x has"): paged.append(c, b, wide, P, 4, named)
    with pytest.raises(TypeError, match="q has"): paged.append(c, b, P, wide, 4, "float16", q_dtype=named)
    with pytest.raises(TypeError, match="q has"): paged.attention(c, b, wide, P, 4, named)
    with pytest.raises(TypeError, match="out has"): paged.attention(c, b, P, wide, 4, out_dtype=named)
    with pytest.raises(TypeError, match="x has"): paged.head_norm_rope(wide, P, 2, 4, 2, 64, named)
    with pytest.raises(TypeError, match="out has"): paged.head_norm_rope(P, wide, 2, 4, 2, 64, out_dtype=named)
  for named, given in (("float16", np.float16), ("bfloat16", np.uint16), ("float32", np.float32)): paged.PagedCache(4, 16, 2, 64, named, k=pool(given), v=pool(given))
  paged.PagedCache(2, 16, 2, 64, "bfloat16", k=Fake((2, 2, 16, 64, 2), np.uint8), v=P)


def test_tensors_that_are_not_laid_out_as_the_call_says(lib):
  """Foreign tensors on the host, and those whose values lie apart without a stride that says so."""
  import torch
  class OnDevice:      # (a host tensor that passes for one of the device)
    is_cuda = True
    def __init__(self, t): self.t = t
    def __getattr__(self, name): return getattr(self.t, name)
  c, b = paged.PagedCache(4, 16, 2, 64, k=P, v=P), paged.PagedBatch(*(Fake(s, np.int32) for s in ((3,), (2,), (2, 5))), 2, 1, 9)
  apart = OnDevice(torch.zeros(2, 1024)[:, :512])
  with pytest.raises(ValueError, match="stride"): paged.append(c, b, apart, P, 4)
  with pytest.raises(ValueError, match="stride"): paged.append(c, b, P, apart, 4)
  with pytest.raises(ValueError, match="stride"): paged.attention(c, b, apart, P, 4)
  with pytest.raises(ValueError, match="stride"): paged.attention(c, b, P, apart, 4)
  with pytest.raises(ValueError, match="stride"): paged.head_norm_rope(apart, P, 2, 4, 2, 64)
  with pytest.raises(ValueError, match="stride"): paged.head_norm_rope(P, apart, 2, 4, 2, 64)
  with pytest.raises(ValueError, match="contiguous"): paged.head_norm_rope(P, P, 2, 4, 2, 64, rope=Fake((9, 64), np.float32), positions=OnDevice(torch.zeros(4, dtype=torch.int32)[::2]))
  with pytest.raises(ValueError, match="contiguous"): paged.append(c, b, P, P, 4, q_norm=OnDevice(torch.zeros(128, dtype=torch.float16)[::2]))
  half = torch.zeros(4, 2, 16, 128, dtype=torch.float16)
  with pytest.raises(ValueError, match="contiguous"): paged.PagedCache(4, 16, 2, 64, k=OnDevice(half[..., :64]), v=OnDevice(half[..., 64:]))
  paged.PagedCache(4, 16, 2, 64, k=OnDevice(half[..., :64]), v=OnDevice(half[..., 64:]), strides=(2 * 16 * 128, 16 * 128, 128))
  for call in (lambda x: paged.append(c, b, x, P, 4), lambda x: paged.append(c, b, P, x, 4), lambda x: paged.attention(c, b, P, x, 4), lambda x: paged.head_norm_rope(x, P, 2, 4, 2, 64),
               lambda x: paged.PagedCache(1, 1, 1, 16, "float32", k=x, v=P), lambda x: paged.PagedBatch(Fake((3,), np.int32), torch.zeros(2, dtype=torch.int32), Fake((2, 5), np.int32), 2, 1, 9)):
    with pytest.raises(ValueError, match="host"): call(torch.zeros(2, 512))


class Workspaces:
  """The library without a device: memory is numbers, and what is done to it is written down."""
  def __init__(self, lib): self.lib, self.log, self.fail, self.capturing = lib, [], False, 0
  def __getattr__(self, name): return getattr(self.lib, name)
  def b200q_pool_alloc(self, p, nbytes, stream):
    p._obj.value = 0x10000 * (1 + len(self.log))
    self.log.append(("alloc", p._obj.value, stream))
    return 0
  def b200q_pool_free(self, ptr): return 0
  def b200q_memset(self, ptr, value, nbytes, stream):
    self.log.append(("memset", ptr, stream or 0))
    return -5 if self.fail else 0
  def b200q_device_synchronize(self):
    self.log.append(("wait",))
    return 0
  def b200q_stream_is_capturing(self, stream, flag):
    flag._obj.value = self.capturing
    return 0


@pytest.fixture
def workspaces(lib, monkeypatch):
  w = Workspaces(lib)
  monkeypatch.setattr(_lib, "load", lambda: w)
  monkeypatch.setattr(paged, "_entry", {**{n: getattr(lib, n) for n in ("b200q_paged_attention_workspace_bytes",)}, "b200q_paged_attention": lambda *a: 0, "b200q_paged_append": lambda *a: 0})
  return w


def a_batch(): return paged.PagedBatch(*(Fake(s, np.int32) for s in ((3,), (2,), (2, 500))), 2, 1, 8000)


def test_a_workspace_that_could_not_be_zeroed_is_not_kept(workspaces):
  """Counters that are not zero would make later calls leave rows out: a reservation that failed is made anew."""
  c, b = paged.PagedCache(4, 16, 2, 64, k=P, v=P), a_batch()
  workspaces.fail = True
  with pytest.raises(_lib.B200QError): paged.attention(c, b, P, P, 4)
  workspaces.fail = False
  paged.attention(c, b, P, P, 4)
  kinds = [e[0] for e in workspaces.log if e[0] != "wait"]
  assert kinds == ["alloc", "memset"] * 2 and workspaces.log[-1 if workspaces.log[-1][0] == "memset" else -2][1] == b._ws.ptr
  paged.attention(c, b, P, P, 4)
  assert [e[0] for e in workspaces.log if e[0] != "wait"] == kinds


def test_a_captured_call_is_reserved_beforehand(workspaces):
  c, b = paged.PagedCache(4, 16, 2, 64, k=P, v=P), a_batch()
  workspaces.capturing = 1
  with pytest.raises(RuntimeError, match="reserve"): paged.attention(c, b, P, P, 4, stream=7)
  assert not workspaces.log
  workspaces.capturing = 0
  b.reserve(c, 4)
  workspaces.capturing = 1
  paged.attention(c, b, P, P, 4, stream=7)


def test_a_graph_keeps_what_its_paged_calls_use(workspaces, monkeypatch):
  """The caches and batches (tables, workspaces) of captured calls live as long as the graph; calls on other streams, or behind the capture, are nothing to it."""
  import gc, weakref
  from tinygrad_b200.runtime import Graph, Stream
  monkeypatch.setattr(Workspaces, "b200q_graph_begin", lambda self, s: 0, raising=False)
  monkeypatch.setattr(Workspaces, "b200q_graph_end", lambda self, s, p: 0, raising=False)
  made = [(paged.PagedCache(4, 16, 2, 64, k=P, v=P), a_batch()) for _ in range(4)]
  for c, b in made: b.reserve(c, 4)
  stream = Stream(7)
  graph = Graph(stream)
  with graph:
    paged.attention(*made[0], P, P, 4, stream=stream)
    paged.append(*made[1], P, 2 * P, 4, stream=7)
    paged.attention(*made[2], P, P, 4, stream=Stream(9))
  paged.attention(*made[3], P, P, 4, stream=stream)
  seen = [(weakref.ref(c), weakref.ref(b)) for c, b in made]
  del made, c, b
  gc.collect()
  assert [(c() is not None, b() is not None) for c, b in seen] == [(True, True)] * 2 + [(False, False)] * 2
  del graph
  gc.collect()
  assert not any(b() for _, b in seen)


def test_a_capture_that_fails_keeps_nothing_open(workspaces, monkeypatch):
  from tinygrad_b200.runtime import Graph, Stream
  monkeypatch.setattr(Workspaces, "b200q_graph_begin", lambda self, s: 0, raising=False)
  monkeypatch.setattr(Workspaces, "b200q_graph_end", lambda self, s, p: -5, raising=False)
  with pytest.raises(_lib.B200QError):
    with Graph(Stream(7)): pass
  with pytest.raises(KeyError):
    with Graph(Stream(7)): raise KeyError
  assert not Graph.open


def test_a_first_call_zeroes_its_workspace_on_its_own_stream(workspaces):
  """No wait for the device: a batch may live as briefly as a step.  One that is reserved beforehand is ready for any stream."""
  c, b = paged.PagedCache(4, 16, 2, 64, k=P, v=P), a_batch()
  paged.attention(c, b, P, P, 4, stream=7)
  assert workspaces.log == [("alloc", b._ws.ptr, 7), ("memset", b._ws.ptr, 7)]
  b = a_batch()
  del workspaces.log[:]
  b.reserve(c, 4)
  assert workspaces.log == [("alloc", b._ws.ptr, 0), ("memset", b._ws.ptr, 0), ("wait",)]
  b.reserve(c, 4)
  assert len(workspaces.log) == 3


@pytest.mark.parametrize("change", [dict(out_dtype=F16), dict(q_stride=512), dict(out_stride=320), dict(q_dtype=BF16)])
def test_attention_in_place_of_other_rows_is_refused(lib, change):
  """out may be q itself; with other types or strides a row would be written where another is still to be read."""
  a = _lib.PagedAttnArgs(P, P, F32, F32, 0, 0, 4, 0.0, P, 1 << 30)
  for k, v in change.items(): setattr(a, k, v)
  assert call(lib.b200q_paged_attention, cache(), batch(), a) == -1


def test_tables_of_different_kinds(lib):
  """A batch's tables may be buffers and foreign tensors in any mixture; each has to be contiguous."""
  import torch
  class OnDevice:
    is_cuda = True
    def __init__(self, t): self.t = t
    def __getattr__(self, name): return getattr(self.t, name)
  i = lambda *s: OnDevice(torch.zeros(s, dtype=torch.int32))
  f = lambda *s: Fake(s, np.int32)
  for row_off, length, pages in ((i(3), f(2), f(2, 5)), (f(3), i(2), f(2, 5)), (f(3), f(2), i(2, 5)), (i(3), i(2), i(2, 5))): paged.PagedBatch(row_off, length, pages, 2, 1, 9)
  apart = lambda *s: OnDevice(torch.zeros(*s[:-1], 2 * s[-1], dtype=torch.int32)[..., ::2])
  for row_off, length, pages in ((apart(3), f(2), f(2, 5)), (f(3), apart(2), f(2, 5)), (f(3), f(2), apart(2, 5)), (i(3), apart(2), i(2, 5))):
    with pytest.raises(ValueError, match="contiguous"): paged.PagedBatch(row_off, length, pages, 2, 1, 9)


def test_page_locked_tensors_are_the_device_s_to_read(lib):
  """The device reaches page-locked host memory: tables may stand there."""
  import torch
  class Pinned:
    is_cuda, is_pinned = False, lambda self: True
    def __init__(self, t): self.t = t
    def __getattr__(self, name): return getattr(self.t, name)
  length = Pinned(torch.zeros(2, dtype=torch.int32))
  assert paged.PagedBatch(Fake((3,), np.int32), length, Fake((2, 5), np.int32), 2, 1, 9).desc.length == length.data_ptr()
