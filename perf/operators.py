"""The paged-cache operators as cases that can be timed: appending a batch's keys and values to pages (with the norms of the heads and the position
rotation on the way), the norms and the rotation alone, and attention of new tokens over the pages.

A case is a dict of plain values.  `prepare` makes what a serving program holds before the call: the projections of the new tokens, the pages with
the earlier tokens' keys and values, the tables that say which sequence has which pages.  `run` is one call: in its plain form (`own` false) elementary
torch operations in 32 bits, else the package's own entry points.

A batch is ragged: sequence i has new[i] tokens that are computed now, at the end of its len[i] tokens."""
import math
import random
import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-6
THETA = 500000.0


def listed():
  return [
    # ---- appending: a chat turn's next token, the smallest call there is
    dict(name="append-1", kind="append", seqs=1, new=1, ctx=513, heads=32, kv_heads=8, dim=128, page=16, rope=128, x="float32", cache="float16", norms=False, mix=0),
    # one token of each of 64 sequences of different lengths, heads normed
    dict(name="append-64-normed", kind="append", seqs=64, new=1, ctx=2048, heads=28, kv_heads=4, dim=128, page=64, rope=128, x="float32", cache="float16", norms=True, mix=3),
    # a long prompt's chunk, heads normed
    dict(name="append-4096-normed", kind="append", seqs=1, new=4096, ctx=6000, heads=32, kv_heads=8, dim=128, page=16, rope=128, x="float32", cache="float16", norms=True, mix=0),
    # several prompts together, narrow heads, half of each head rotated
    dict(name="append-ragged-bf16", kind="append", seqs=9, new=1500, ctx=2500, heads=16, kv_heads=16, dim=64, page=32, rope=32, x="bfloat16", cache="bfloat16", norms=False, mix=5),
    # ---- the norms (and the rotation) alone, for caches that are not paged: one token, a prompt
    dict(name="norm-1", kind="norm", rows=1, ctx=2048, heads=32, kv_heads=8, dim=128, rope=128, x="float32"),
    dict(name="norm-8191-f16", kind="norm", rows=8191, ctx=8192, heads=28, kv_heads=4, dim=128, rope=0, x="float16"),
    # ---- attention: a chat turn's next token
    dict(name="attend-1", kind="attend", seqs=1, new=1, ctx=513, heads=32, kv_heads=8, dim=128, page=16, x="float32", cache="float16", mix=0),
    # serving: one token of each of 48 sequences of different lengths, 7 heads to a key head
    dict(name="attend-48-ragged", kind="attend", seqs=48, new=1, ctx=8192, heads=28, kv_heads=4, dim=128, page=64, x="float32", cache="float16", mix=7),
    # one very long conversation
    dict(name="attend-long-f16", kind="attend", seqs=1, new=1, ctx=131071, heads=32, kv_heads=8, dim=128, page=32, x="float16", cache="float16", mix=0),
    # a chunk of a long prompt behind as many cached tokens
    dict(name="attend-chunk-f16", kind="attend", seqs=1, new=4096, ctx=8192, heads=32, kv_heads=8, dim=128, page=16, x="float16", cache="float16", mix=0),
    # the same with the 32-bit rows that the package's own models carry
    dict(name="attend-chunk-f32", kind="attend", seqs=2, new=1000, ctx=2300, heads=32, kv_heads=8, dim=128, page=128, x="float32", cache="float16", mix=9),
    # prompts and single tokens in one batch, narrow heads
    dict(name="attend-mixed-bf16", kind="attend", seqs=12, new=700, ctx=3000, heads=16, kv_heads=4, dim=64, page=16, x="bfloat16", cache="bfloat16", mix=11),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  kind = rng.choice(["append", "append", "norm", "attend", "attend", "attend", "attend"])
  heads, kv_heads = rng.choice([(32, 8), (28, 4), (16, 16), (8, 2), (16, 4)])
  x = rng.choice(["float32", "float16", "bfloat16"])
  dim = rng.choice([64, 128, 128])
  if kind == "norm":
    return dict(kind=kind, rows=_log(rng, 1, 8191), ctx=rng.choice([2048, 8192]), heads=heads, kv_heads=kv_heads, dim=dim, rope=rng.choice([0, dim, dim // 2]), x=x)
  case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]), x=x, cache="float16" if x != "bfloat16" else "bfloat16",
              mix=rng.randrange(1 << 20))
  if kind == "append":
    seqs = _log(rng, 1, 64)
    new = _log(rng, 1, max(1, 4096 // seqs))
    return dict(case, seqs=seqs, new=new, ctx=new + _log(rng, 1, 2000), rope=rng.choice([dim, dim, dim // 2]), norms=rng.random() < 0.5)
  if rng.random() < 0.5:      # single tokens, or a few
    seqs = _log(rng, 1, 64)
    return dict(case, seqs=seqs, new=rng.choice([1, 1, 1, 2, 4]), ctx=_log(rng, 33, max(64, min(131071, 400000 // seqs))))
  seqs = _log(rng, 1, 12)
  new = _log(rng, 5, max(6, 2048 // seqs))
  return dict(case, seqs=seqs, new=new, ctx=new + _log(rng, 1, 4096))


def batch_of(case):
  """(new tokens, all tokens) of each sequence; the first has the largest of both."""
  r, new, ctx = random.Random(case["mix"]), case["new"], case["ctx"]
  got = [(new, ctx)]
  for _ in range(case["seqs"] - 1):
    n = _log(r, 1, new)
    got.append((n, r.randint(n, ctx)))
  return [n for n, _ in got], [l for _, l in got]


def _rand(g, shape, dtype, scale=1.0):
  return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _table(rows, dim):
  """cos || sin of every position, as the package's models keep it."""
  f = THETA ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
  a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * f
  return torch.cat([a.cos(), a.sin()], -1).float()


def prepare(case, seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  h, hk, d, xt = case["heads"], case["kv_heads"], case["dim"], TYPES[case["x"]]
  s = {"case": case}
  if case["kind"] == "norm":
    n = case["rows"]
    s["x"] = _rand(g, (n, (h + 2 * hk) * d), xt, 1.7)
    s["out"] = torch.empty((n, (h + hk) * d), dtype=xt, device="cuda")
    s["positions"] = torch.randint(0, case["ctx"], (n,), generator=g, device="cuda", dtype=torch.int32)
  else:
    new, length = batch_of(case)
    n, ps = sum(new), case["page"]
    pages = [-(-l // ps) for l in length]
    order = torch.randperm(sum(pages) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((case["seqs"], max(pages)), dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(pages):
      table[i, :p] = order[at:at + p]
      at += p
    s["table"], ct = table, TYPES[case["cache"]]
    s["row_off"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    s["length"] = torch.tensor(length, device="cuda", dtype=torch.int32)
    shape = (sum(pages) + 3, hk, ps, d)
    s["k"], s["v"] = _rand(g, shape, ct, 1.3), _rand(g, shape, ct)
    if case["kind"] == "append":
      s["x"] = _rand(g, (n, (h + 2 * hk) * d), xt, 1.7)
    else:
      s["x"] = _rand(g, (n, h * d), xt, 1.3)
    s["out"] = torch.empty((n, h * d), dtype=xt, device="cuda")
  if case.get("rope"): s["rope"] = _table(case["ctx"], case["rope"])
  if case.get("norms", case["kind"] == "norm"):
    s["q_norm"], s["k_norm"] = (1 + _rand(g, (d,), torch.float32, 0.2)).half(), (1 + _rand(g, (d,), torch.float32, 0.2)).half()
  if own:      # the handles a program keeps: where the pages are, and which sequence has which
    from tinygrad_b200 import paged
    if case["kind"] != "norm":
      s["pages"] = paged.PagedCache(s["k"].shape[0], ps, hk, d, case["cache"], k=s["k"], v=s["v"])
      s["batch"] = paged.PagedBatch(s["row_off"], s["length"], s["table"], n_rows=n, max_new=case["new"], max_len=case["ctx"])
      if case["kind"] == "attend": s["batch"].reserve(s["pages"], h, case["x"])
  return s


def _normed(x, w):
  return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _rotated(x, table):
  """x [n, heads, dim], table [n, rotated dimensions]."""
  if table is None: return x
  r = table.shape[-1] // 2
  cos, sin, a, b = table[:, None, :r], table[:, None, r:], x[..., :r], x[..., r:2 * r]
  return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * r:]], -1)


def _places(s):
  """Of every new row: its sequence, its number in there, its position."""
  off, rows = s["row_off"].long(), torch.arange(s["x"].shape[0], device="cuda")
  seq = torch.searchsorted(off[1:], rows, right=True)
  i = rows - off[seq]
  return seq, i, s["length"].long()[seq] - (off[seq + 1] - off[seq]) + i


def run(s):
  return {"append": _append, "norm": _norm, "attend": _attend}[s["case"]["kind"]](s)


def _append(s):
  c = s["case"]
  h, hk, d = c["heads"], c["kv_heads"], c["dim"]
  if own:
    from tinygrad_b200 import paged
    paged.append(s["pages"], s["batch"], s["x"], s["out"], h, c["x"], rope=s["rope"], q_norm=s.get("q_norm"), k_norm=s.get("k_norm"), norm_eps=EPS)
    return {"q": s["out"], "k": s["k"], "v": s["v"]}
  seq, _, pos = _places(s)
  x = s["x"].float().view(-1, h + 2 * hk, d)
  table = s["rope"][pos]
  q, k = _rotated(_normed(x[:, :h], s.get("q_norm")), table), _rotated(_normed(x[:, h:h + hk], s.get("k_norm")), table)
  page, slot = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
  s["k"][page, :, slot] = k.to(s["k"].dtype)
  s["v"][page, :, slot] = x[:, h + hk:].to(s["v"].dtype)
  return {"q": q.reshape(-1, h * d).to(s["x"].dtype), "k": s["k"], "v": s["v"]}


def _norm(s):
  c = s["case"]
  h, hk, d = c["heads"], c["kv_heads"], c["dim"]
  if own:
    from tinygrad_b200 import paged
    paged.head_norm_rope(s["x"], s["out"], c["rows"], h, hk, d, c["x"], q_norm=s["q_norm"], k_norm=s["k_norm"], norm_eps=EPS, rope=s.get("rope"), positions=s["positions"],
                         x_stride=(h + 2 * hk) * d)
    return s["out"]
  x = s["x"].float().view(-1, h + 2 * hk, d)
  table = s["rope"][s["positions"].long()] if "rope" in s else None
  q, k = _rotated(_normed(x[:, :h], s["q_norm"]), table), _rotated(_normed(x[:, h:h + hk], s["k_norm"]), table)
  return torch.cat([q, k], 1).reshape(-1, (h + hk) * d).to(s["x"].dtype)


def _attend(s):
  c = s["case"]
  h, hk, d = c["heads"], c["kv_heads"], c["dim"]
  if own:
    from tinygrad_b200 import paged
    paged.attention(s["pages"], s["batch"], s["x"], s["out"], h, c["x"])
    return s["out"]
  seq, i, pos = _places(s)
  n_seqs, new, keys = c["seqs"], c["new"], s["table"].shape[1] * c["page"]
  q = torch.zeros((n_seqs, new, hk, h // hk, d), device="cuda")
  q[seq, i] = s["x"].float().view(-1, hk, h // hk, d)
  last = torch.full((n_seqs, new), -1, device="cuda", dtype=torch.long)
  last[seq, i] = pos
  k, v = (s[p][s["table"].long()].transpose(1, 2).reshape(n_seqs, hk, keys, d).float() for p in "kv")
  w = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(n_seqs, hk, -1, d), k.transpose(-1, -2)).view(n_seqs, hk, h // hk, new, keys) * d ** -0.5
  w = w.masked_fill_((torch.arange(keys, device="cuda") > last[..., None])[:, None, None], -math.inf)
  top = w.amax(-1, keepdim=True)
  w = w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
  total = w.sum(-1, keepdim=True)
  o = torch.matmul(w.view(n_seqs, hk, -1, keys), v).view(n_seqs, hk, h // hk, new, d) / torch.where(total == 0, 1.0, total)
  return o.permute(0, 3, 1, 2, 4)[seq, i].reshape(-1, h * d).to(s["x"].dtype)


def work(case):
  h, hk, d = case["heads"], case["kv_heads"], case["dim"]
  xs = 4 if case["x"] == "float32" else 2
  if case["kind"] == "norm":
    n = case["rows"] * (h + hk) * d
    return {"bytes": 2 * n * xs + 4 * d + (case["rows"] * 4 + min(case["rows"], case["ctx"]) * case["rope"] * 4 if case["rope"] else 0), "flops": 8 * n}
  new, length = batch_of(case)
  n = sum(new)
  if case["kind"] == "append":
    positions = min(n, case["ctx"])
    return {"bytes": n * (h + 2 * hk) * d * xs + n * h * d * xs + n * 2 * hk * d * 2 + positions * case["rope"] * 4, "flops": 8 * n * (h + hk) * d}
  pairs = sum(a * (l - a) + a * (a + 1) // 2 for a, l in zip(new, length))
  return {"bytes": sum(length) * 2 * hk * d * 2 + 2 * n * h * d * xs, "flops": 4 * h * d * pairs}


def exact(case, seed):
  """The definition, row by row or head by head, in 64 bits."""
  s = prepare(case, seed)
  h, hk, d = case["heads"], case["kv_heads"], case["dim"]

  def head(x, w, at):
    x = x.double()
    if w is not None: x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
    if "rope" in s:
      r, y = case["rope"] // 2, x.clone()
      z = torch.complex(x[..., :r], x[..., r:2 * r]) * torch.complex(s["rope"][at, :r].double(), s["rope"][at, r:].double())[:, None]
      y[..., :r], y[..., r:2 * r] = z.real, z.imag
      x = y
    return x

  if case["kind"] == "norm":
    rows, at = s["x"].view(case["rows"], -1, d), s["positions"].long()
    return torch.cat([head(rows[:, :h], s["q_norm"], at), head(rows[:, h:h + hk], s["k_norm"], at)], 1).reshape(case["rows"], -1)
  new, length = batch_of(case)
  ps, got = case["page"], []
  k, v = s["k"].double(), s["v"].double()
  start = 0
  for i, (n, l) in enumerate(zip(new, length)):
    x = s["x"][start:start + n].view(n, -1, d)
    start += n
    where = torch.arange(l, device="cuda")
    page, slot = s["table"][i][where // ps].long(), where % ps
    if case["kind"] == "append":
      at = where[l - n:]
      got.append(head(x[:, :h], s.get("q_norm"), at).reshape(n, -1))
      kx, vx = head(x[:, h:h + hk], s.get("k_norm"), at), x[:, h + hk:].double()
      for j in range(hk): k[page[l - n:], j, slot[l - n:]], v[page[l - n:], j, slot[l - n:]] = kx[:, j], vx[:, j]
      continue
    out = torch.empty((n, h, d), dtype=torch.float64, device="cuda")
    hidden = where[None, :] > where[l - n:, None]
    for j in range(h):
      kk, vv = k[page, j // (h // hk), slot], v[page, j // (h // hk), slot]
      out[:, j] = torch.softmax((x[:, j].double() @ kk.T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1) @ vv
    got.append(out.reshape(n, -1))
  q = torch.cat(got)
  return {"q": q, "k": k, "v": v} if case["kind"] == "append" else q
