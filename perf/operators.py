"""The sequence and loss operators over embedding rows, as they are measured: attention over ragged
rows (the pooled form with one query per row and the many-query form, each forward and with its
gradient), attention over a prefix that the whole batch shares, and the softmax cross entropy over
the rows of a table with its gradient.

`run` computes them in elementary torch operations, in 32 bits, rounded once at the end, or, where
`own` is true, calls the framework's operators."""
import math
import random

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------- the cases
def listed():
  return [
      # one request's behaviour slots pooled by the candidate: a few dozen short rows, latency only
      {"name": "pool_request", "op": "pool", "grad": False, "dtype": "fp32", "batch": 33, "least": 0,
       "most": 100, "heads": 1, "kv_heads": 1, "dim": 16, "mask": False},
      # a training batch of one multi-hot slot (about 50 ids a row, a long tail) pooled by attention
      {"name": "pool_train", "op": "pool", "grad": True, "dtype": "fp32", "batch": 16384, "least": 0,
       "most": 300, "heads": 1, "kv_heads": 1, "dim": 32, "mask": True},
      # few users with histories of a lifetime, one token each: the long axis has to be split
      {"name": "pool_lifelong", "op": "pool", "grad": False, "dtype": "bf16", "batch": 7, "least": 9000,
       "most": 120000, "heads": 4, "kv_heads": 2, "dim": 64, "mask": False},
      # self attention over the first N of a slot's ids in a sequential recommender's training step,
      # ids that the table does not hold masked, small rows in 32 bits
      {"name": "seq_train_rows", "op": "seq", "grad": True, "dtype": "fp32", "batch": 301, "least": 0,
       "most": 200, "heads": 4, "kv_heads": 2, "dim": 32, "mask": True, "causal": True},
      # the same with a transformer's widths
      {"name": "seq_train", "op": "seq", "grad": True, "dtype": "bf16", "batch": 96, "least": 100,
       "most": 2048, "heads": 8, "kv_heads": 8, "dim": 64, "mask": False, "causal": True},
      # encoding a few long histories once, for serving
      {"name": "seq_encode", "op": "seq", "grad": False, "dtype": "bf16", "batch": 6, "least": 1000,
       "most": 8192, "heads": 8, "kv_heads": 2, "dim": 128, "mask": False, "causal": True},
      # a handful of candidates against one short history
      {"name": "prefix_request", "op": "prefix", "dtype": "fp32", "prefix": 300, "batch": 17, "tokens": 1,
       "most": 0, "heads": 2, "kv_heads": 2, "dim": 16},
      # a ranking request: two thousand candidates of up to three tokens behind one user's history
      {"name": "prefix_rank", "op": "prefix", "dtype": "bf16", "prefix": 8192, "batch": 2000, "tokens": 3,
       "most": 3, "heads": 8, "kv_heads": 2, "dim": 64},
      # a step of few candidates behind a prefix so long that reading it is the work
      {"name": "prefix_lifelong", "op": "prefix", "dtype": "bf16", "prefix": 200001, "batch": 61, "tokens": 1,
       "most": 40, "heads": 16, "kv_heads": 4, "dim": 128},
      # in-batch softmax of a two-tower model, corrected by the sampling frequency, small batch
      {"name": "ce_batch", "op": "ce", "grad": True, "dtype": "fp32", "rows": 1000, "vocab": 1000, "dim": 16,
       "bias": True},
      # sampled softmax of a training step against table rows in 32 bits
      {"name": "ce_sampled", "op": "ce", "grad": True, "dtype": "fp32", "rows": 8192, "vocab": 16385, "dim": 64,
       "bias": True},
      # the full softmax over a catalogue of a million rows
      {"name": "ce_catalogue", "op": "ce", "grad": True, "dtype": "bf16", "rows": 4096, "vocab": 1000003,
       "dim": 64, "bias": False},
  ]


def _between(rng, lo, hi):
  """A whole number spread over the logarithm of [lo, hi]."""
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  op = rng.choice(["pool", "seq", "prefix", "ce"])
  kv = rng.choice([1, 2, 4])
  group = rng.choice([1, 1, 2, 4])
  dtype = rng.choice(["fp32", "bf16"])
  dim = rng.choice([8, 16, 24, 32, 48, 64, 96, 128])
  if op == "pool":
    batch = _between(rng, 1, 20000)
    most = max(4, min(_between(rng, 4, 100000), 1000000 // batch))
    return {"op": op, "grad": rng.random() < 0.5, "dtype": dtype, "batch": batch, "least": rng.randrange(0, 3),
            "most": most, "heads": kv * group, "kv_heads": kv, "dim": min(dim, 64), "mask": rng.random() < 0.5}
  if op == "seq":
    most = _between(rng, 4, 4000)
    batch = _between(rng, 1, max(1, min(500, int(4e8 / (most * most * kv * group)))))
    return {"op": op, "grad": rng.random() < 0.6, "dtype": dtype, "batch": batch, "least": rng.randrange(0, 3),
            "most": most, "heads": kv * group, "kv_heads": kv, "dim": dim, "mask": rng.random() < 0.5,
            "causal": rng.random() < 0.7}
  if op == "prefix":
    tokens = rng.choice([1, 1, 2, 5])
    batch = _between(rng, 1, 1500)
    prefix = _between(rng, 16, min(150000, int(4e8 / (batch * tokens * kv * group))))
    return {"op": op, "dtype": dtype, "prefix": prefix, "batch": batch, "tokens": tokens,
            "most": rng.choice([0, tokens, tokens + 11]), "heads": kv * group, "kv_heads": kv, "dim": dim}
  rows = _between(rng, 1, 8192)
  vocab = _between(rng, 2, min(1000000, int(4e8 / rows)))
  return {"op": op, "grad": rng.random() < 0.7, "dtype": dtype, "rows": rows, "vocab": vocab, "dim": dim,
          "bias": rng.random() < 0.5}


def _lengths(case):
  """The lengths of a case's rows, as a set: log-uniform, so most rows are short and a few are long.
  They come from the sizes alone (`work` counts them); their order comes from the seed."""
  rng = random.Random(case["batch"] * 1000003 + case["most"])
  lo, hi = case["least"], case["most"]
  lens = [min(hi, int(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1.5)))) - 1 + (lo > 0))
          for _ in range(case["batch"])]
  lens[0] = hi
  return [max(lo, n) for n in lens]


def _candidate_lengths(case):
  """(query tokens, own keys) of every candidate behind a prefix."""
  rng = random.Random(case["batch"] * 1000003 + case["prefix"])
  lq = [rng.randint(1, case["tokens"]) for _ in range(case["batch"])]
  if not case["most"]:
    return lq, [0] * len(lq)
  return lq, [max(n, rng.randint(0, case["most"])) if case["tokens"] > 1 else rng.randint(0, case["most"])
              for n in lq]


# ------------------------------------------------------------------------------- the inputs
def _splits(lens):
  out = [0]
  for n in lens:
    out.append(out[-1] + n)
  return torch.tensor(out, dtype=torch.int64, device="cuda")


def prepare(case, seed):
  gen = torch.Generator(device="cuda").manual_seed(seed)
  dtype = _TYPES[case["dtype"]]

  def normal(*shape, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

  d = case["dim"]
  s = {"case": case}
  if case["op"] == "ce":
    n, v = case["rows"], case["vocab"]
    # logits of standard deviation 2: scores that a trained model has begun to tell apart
    s["query"] = normal(n, d, scale=math.sqrt(2.0) / d ** 0.25)
    s["rows"] = normal(v, d, scale=math.sqrt(2.0) / d ** 0.25)
    s["labels"] = torch.randint(0, v, (n,), generator=gen, device="cuda")
    s["labels"][torch.rand(n, generator=gen, device="cuda") < 0.05] = -1  # rows without a label
    # log of the steps between two occurrences of a candidate: what corrects for its frequency
    s["bias"] = (torch.rand(v, generator=gen, device="cuda") * 6.0) if case["bias"] else None
    s["weight"] = torch.rand(n, generator=gen, device="cuda") + 0.5  # every sample's weight
    return s
  h, kv = case["heads"], case["kv_heads"]
  order = random.Random(seed)
  if case["op"] == "prefix":
    lq, lk = _candidate_lengths(case)
    perm = list(range(len(lq)))
    order.shuffle(perm)
    lq, lk = [lq[i] for i in perm], [lk[i] for i in perm]
    s["prefix_key"], s["prefix_value"] = normal(case["prefix"], kv, d), normal(case["prefix"], kv, d)
    s["key"], s["value"] = (normal(sum(lk), kv, d), normal(sum(lk), kv, d)) if case["most"] else (None, None)
    s["key_splits"] = _splits(lk) if case["most"] else None
    s["query_splits"] = _splits(lq) if case["tokens"] > 1 else None
    s["lq"], s["lk"] = lq, lk
    s["query"] = normal(sum(lq), h, d)
    return s
  lens = _lengths(case)
  order.shuffle(lens)
  n = sum(lens)
  s["lens"], s["key_splits"] = lens, _splits(lens)
  nq = case["batch"] if case["op"] == "pool" else n
  s["query"], s["key"] = normal(nq, h, d), normal(n, kv, d)
  # pooling weighs and sums the same embeddings; a sequence layer has projected values
  s["value"] = None if case["op"] == "pool" else normal(n, kv, d)
  # ids that the table does not hold
  s["mask"] = torch.rand(n, generator=gen, device="cuda") > 0.1 if case["mask"] else None
  if case["grad"]:
    s["grad"] = normal(nq, h, d)
  return s


# ------------------------------------------------------------------------------- the plain forms
def _pad_index(splits, most):
  """[batch, most] positions of the padded form of ragged rows, and which of them exist."""
  at = splits[:-1, None] + torch.arange(most, device=splits.device)[None]
  there = at < splits[1:, None]
  return torch.where(there, at, torch.zeros_like(at)), there


def _pad(x, at, there):
  """[n, heads, d] -> [batch, heads, most, d] in 32 bits, zeros where nothing is."""
  if not x.shape[0]:
    return x.new_zeros((at.shape[0], x.shape[1], at.shape[1], x.shape[2]), dtype=torch.float32)
  return (x[at].float() * there[..., None, None]).transpose(1, 2).contiguous()


def _products(a, b):
  return torch.matmul(a, b.contiguous())


def _softmax(logits, keep):
  logits = torch.where(keep, logits, torch.full_like(logits, -math.inf))
  top = logits.amax(-1, keepdim=True)
  top = torch.where(top == -math.inf, torch.zeros_like(top), top)
  e = torch.exp(logits - top)
  total = e.sum(-1, keepdim=True)
  return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_attention(s):
  case = s["case"]
  h, kv, d = case["heads"], case["kv_heads"], case["dim"]
  group = h // kv
  shared = s["value"] is None
  most = max(s["lens"] + [1])
  at, there = _pad_index(s["key_splits"], most)
  k = _pad(s["key"], at, there)
  v = k if shared else _pad(s["value"], at, there)
  batch = at.shape[0]
  keep = there if s["mask"] is None else there & (s["mask"][at] if s["mask"].numel() else there)
  keep = keep[:, None, None, :]
  if case["op"] == "pool":
    nq = 1
    q = s["query"].float().view(batch, h, 1, d)
  else:
    nq = most
    q = _pad(s["query"], at, there)
    if case["causal"]:
      pos = torch.arange(most, device=k.device)
      keep = keep & (pos[None, :] <= pos[:, None])
  # the query heads of one key head, side by side
  q = q.reshape(batch, kv, group * nq, d)
  keep = keep.expand(batch, 1, nq, most).repeat(1, 1, group, 1)
  scale = 1.0 / math.sqrt(d)
  p = _softmax(_products(q, k.transpose(2, 3)) * scale, keep)
  o = _products(p, v)

  def rows(x, heads, length):  # back to [n, heads, d]
    x = x.view(batch, heads, length, d)
    return x[:, :, 0] if length == 1 and case["op"] == "pool" else x.transpose(1, 2)[there]

  out = rows(o.reshape(batch, h, nq, d), h, nq).to(s["query"].dtype)
  if not case["grad"]:
    return {"out": out}
  if case["op"] == "pool":
    g = s["grad"].float().view(batch, kv, group, d)
  else:
    g = _pad(s["grad"], at, there).reshape(batch, kv, group * nq, d)
  dv = _products(p.transpose(2, 3).contiguous(), g)
  dp = _products(g, v.transpose(2, 3))
  ds = p * (dp - (g * o).sum(-1, keepdim=True)) * scale
  dq = rows(_products(ds, k).reshape(batch, h, nq, d), h, nq)
  dk = _products(ds.transpose(2, 3).contiguous(), q)
  to = s["key"].dtype
  if shared:
    return {"out": out, "dq": dq.to(to), "dk": (dk + dv).transpose(1, 2)[there].to(to)}
  return {"out": out, "dq": dq.to(to), "dk": dk.transpose(1, 2)[there].to(to),
          "dv": dv.transpose(1, 2)[there].to(to)}


def _plain_prefix(s):
  case = s["case"]
  h, kv, d = case["heads"], case["kv_heads"], case["dim"]
  group, nq = h // kv, s["query"].shape[0]
  scale = 1.0 / math.sqrt(d)
  q = s["query"].float().view(nq, kv, group, d).permute(1, 0, 2, 3).contiguous()  # [kv, nq, group, d]
  pk = s["prefix_key"].float().transpose(0, 1).contiguous()  # [kv, prefix, d]
  pv = s["prefix_value"].float().transpose(0, 1).contiguous()
  logits = (_products(q.view(kv, nq * group, d), pk.transpose(1, 2)) * scale).view(kv, nq, group, -1)
  if s["key"] is None:
    p = _softmax(logits, torch.ones((), dtype=torch.bool, device=q.device))
    out = _products(p.view(kv, nq * group, -1), pv).view(kv, nq, group, d)
    return {"out": out.permute(1, 0, 2, 3).reshape(nq, h, d).to(s["query"].dtype)}
  # every token's candidate, its place in it, and the keys of that candidate
  lk = s["key_splits"][1:] - s["key_splits"][:-1]
  tok = torch.arange(nq, device=q.device)
  if s["query_splits"] is None:
    mine, left = tok, torch.zeros_like(tok)
  else:
    mine = (tok[:, None] >= s["query_splits"][None, 1:]).sum(1)
    left = s["query_splits"][1:][mine] - 1 - tok  # tokens of the candidate behind this one
  most = max(s["lk"] + [1])
  at, there = _pad_index(s["key_splits"], most)
  k, v = _pad(s["key"], at, there), _pad(s["value"], at, there)  # [batch, kv, most, d]
  own_logits = (q[:, :, :, None, :] * k[mine].transpose(0, 1)[:, :, None]).sum(-1) * scale  # [kv, nq, group, most]
  keep = torch.arange(most, device=q.device)[None] < (lk[mine] - left)[:, None]
  keep = keep[None, :, None, :].expand(kv, nq, group, most)
  both = torch.cat([torch.ones_like(logits, dtype=torch.bool), keep], -1)
  p = _softmax(torch.cat([logits, own_logits], -1), both)
  n = pk.shape[1]
  out = _products(p[..., :n].reshape(kv, nq * group, n), pv).view(kv, nq, group, d)
  out = out + (p[..., n:, None] * v[mine].transpose(0, 1)[:, :, None]).sum(-2)
  return {"out": out.permute(1, 0, 2, 3).reshape(nq, h, d).to(s["query"].dtype)}


def _plain_ce(s):
  q, w, labels = s["query"].float(), s["rows"].float(), s["labels"]
  logits = _products(q, w.t())
  if s["bias"] is not None:
    logits = logits + s["bias"]
  there = labels >= 0
  label = torch.where(there, labels, torch.zeros_like(labels))
  top = logits.amax(1, keepdim=True)
  hit = logits.gather(1, label[:, None])[:, 0]
  p = torch.exp(logits - top)
  total = p.sum(1, keepdim=True)
  loss = torch.where(there, torch.log(total[:, 0]) + top[:, 0] - hit, torch.zeros_like(hit))
  if not s["case"]["grad"]:
    return {"loss": loss}
  g = s["weight"] * there
  p = p * (g[:, None] / total)
  p[torch.arange(label.shape[0], device=q.device), label] -= g
  out = {"loss": loss, "dquery": _products(p, w).to(s["query"].dtype),
         "drows": _products(p.t().contiguous(), q).to(s["query"].dtype)}
  if s["bias"] is not None:
    out["dbias"] = p.sum(0)
  return out


def _own_run(s):
  from monolith_amd import attention_ops, loss_ops
  case = s["case"]
  if case["op"] == "prefix":
    return {"out": attention_ops.shared_prefix_attention(
        s["query"], s["prefix_key"], s["prefix_value"], s["key"], s["value"], s["key_splits"],
        query_splits=s["query_splits"], causal=s["query_splits"] is not None)}
  if case["op"] == "ce":
    if not case["grad"]:
      return {"loss": loss_ops.softmax_cross_entropy(s["query"], s["rows"], s["labels"], bias=s["bias"])}
    q, w = s["query"].detach().requires_grad_(), s["rows"].detach().requires_grad_()
    leaves, names = [q, w], ["dquery", "drows"]
    bias = s["bias"]
    if bias is not None:
      bias = bias.detach().requires_grad_()
      leaves, names = leaves + [bias], names + ["dbias"]
    loss = loss_ops.softmax_cross_entropy(q, w, s["labels"], bias=bias)
    return {"loss": loss.detach(), **dict(zip(names, torch.autograd.grad(loss, leaves, s["weight"])))}
  q, k, v = s["query"], s["key"], s["value"]
  leaves, names = [], []
  if case["grad"]:
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    leaves, names = [q, k], ["dq", "dk"]
    if v is not None:
      v = v.detach().requires_grad_()
      leaves, names = leaves + [v], names + ["dv"]
  out = attention_ops.ragged_attention(
      q, k, v, s["key_splits"], query_splits=None if case["op"] == "pool" else s["key_splits"],
      key_mask=s["mask"], causal=case.get("causal", False))
  if not case["grad"]:
    return {"out": out}
  return {"out": out.detach(), **dict(zip(names, torch.autograd.grad(out, leaves, s["grad"])))}


def run(state):
  if own:
    return _own_run(state)
  op = state["case"]["op"]
  return _plain_ce(state) if op == "ce" else _plain_prefix(state) if op == "prefix" else _plain_attention(state)


# ------------------------------------------------------------------------------- what they need
def work(case):
  size = 4 if case["dtype"] == "fp32" else 2
  d = case["dim"]
  if case["op"] == "ce":
    n, v = case["rows"], case["vocab"]
    moved = (n + v) * d * size + 8 * n + 4 * n + (4 * v if case["bias"] else 0)
    if not case["grad"]:
      return {"bytes": moved, "flops": 2 * n * v * d}
    return {"bytes": moved + (n + v) * d * size + 4 * n + (4 * v if case["bias"] else 0), "flops": 6 * n * v * d}
  h, kv = case["heads"], case["kv_heads"]
  if case["op"] == "prefix":
    lq, lk = _candidate_lengths(case)
    pairs = sum(lq) * case["prefix"] + sum(a * b - a * (a - 1) // 2 if case["tokens"] > 1 else b
                                           for a, b in zip(lq, lk))
    moved = (2 * sum(lq) * h + 2 * (case["prefix"] + sum(lk)) * kv) * d * size
    moved += 8 * (case["batch"] + 1) * ((case["most"] > 0) + (case["tokens"] > 1))
    return {"bytes": moved, "flops": 4 * d * h * pairs}
  lens = _lengths(case)
  n = sum(lens)
  pool = case["op"] == "pool"
  nq = case["batch"] if pool else n
  pairs = n if pool else sum(x * (x + 1) // 2 if case["causal"] else x * x for x in lens)
  keys = n * kv * (1 if pool else 2)  # elements of a row of keys and values, pooled ones shared
  moved = (2 * nq * h + keys) * d * size + 8 * (case["batch"] + 1) + (n if case["mask"] else 0)
  if not case["grad"]:
    return {"bytes": moved, "flops": 4 * d * h * pairs}
  # the gradient reads the output's gradient and writes those of the inputs; its products are the
  # logits again, the weights' gradient, and one for each of the three inputs
  return {"bytes": moved + (2 * nq * h + keys) * d * size, "flops": 14 * d * h * pairs}


# ------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
  s = prepare(case, seed)
  if case["op"] == "ce":
    return _exact_ce(s)
  if case["op"] == "prefix":
    return _exact_prefix(s)
  return _exact_pool(s) if case["op"] == "pool" else _exact_seq(s)


def _exact_pool(s):
  """Over the ragged rows as they lie: sums by the row that a key belongs to."""
  case = s["case"]
  kv, d, batch = case["kv_heads"], case["dim"], case["batch"]
  group = case["heads"] // kv
  lens = torch.tensor(s["lens"], device="cuda")
  row = torch.repeat_interleave(torch.arange(batch, device="cuda"), lens)
  q = s["query"].double().view(batch, kv, group, d)
  k = s["key"].double()
  score = torch.einsum("nkgd,nkd->nkg", q[row], k) / math.sqrt(d)
  alive = torch.ones(len(row), dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
  e = torch.exp(score.clamp(max=700)) * alive[:, None, None]
  z = torch.zeros(batch, kv, group, dtype=torch.float64, device="cuda").index_add_(0, row, e)
  p = e / z[row].clamp_min(1e-300)
  out = torch.zeros_like(q).index_add_(0, row, p[..., None] * k[:, :, None])
  res = {"out": out.view(batch, -1, d)}
  if case["grad"]:
    g = s["grad"].double().view(batch, kv, group, d)
    dp = torch.einsum("nkgd,nkd->nkg", g[row], k)
    mean = (g * out).sum(-1)
    ds = p * (dp - mean[row]) / math.sqrt(d)
    res["dq"] = torch.zeros_like(q).index_add_(0, row, ds[..., None] * k[:, :, None]).view(batch, -1, d)
    res["dk"] = (ds[..., None] * q[row] + p[..., None] * g[row]).sum(2)
  return res


def _exact_seq(s):
  """One sequence and one head after the other."""
  case = s["case"]
  h, kv, d = case["heads"], case["kv_heads"], case["dim"]
  q, k, v = s["query"].double(), s["key"].double(), s["value"].double()
  out, dq = torch.zeros_like(q), torch.zeros_like(q)
  dk, dv = torch.zeros_like(k), torch.zeros_like(v)
  lo = 0
  for n in s["lens"]:
    hi = lo + n
    if n:
      ok = torch.ones(n, n, dtype=torch.bool, device="cuda")
      if case["causal"]:
        ok = ok.tril()
      if s["mask"] is not None:
        ok = ok & s["mask"][lo:hi]
      for i in range(h):
        j = i // (h // kv)
        score = (q[lo:hi, i] @ k[lo:hi, j].t() / math.sqrt(d)).masked_fill(~ok, -math.inf)
        p = torch.softmax(score, 1).masked_fill(~ok.any(1)[:, None], 0.0)
        out[lo:hi, i] = p @ v[lo:hi, j]
        if case["grad"]:
          g = s["grad"][lo:hi, i].double()
          dp = g @ v[lo:hi, j].t()
          ds = p * (dp - (dp * p).sum(1, keepdim=True)) / math.sqrt(d)
          dv[lo:hi, j] += p.t() @ g
          dq[lo:hi, i] = ds @ k[lo:hi, j]
          dk[lo:hi, j] += ds.t() @ q[lo:hi, i]
    lo = hi
  return {"out": out, "dq": dq, "dk": dk, "dv": dv} if case["grad"] else {"out": out}


def _exact_prefix(s):
  """One candidate after the other for its own keys, head by head for the prefix."""
  case = s["case"]
  h, kv, d = case["heads"], case["kv_heads"], case["dim"]
  q = s["query"].double() / math.sqrt(d)
  out = torch.zeros_like(q)
  own_score = {}
  if s["key"] is not None:
    k, v = s["key"].double(), s["value"].double()
    a = b = 0
    for c, (nq, nk) in enumerate(zip(s["lq"], s["lk"])):
      if nk:
        x = torch.einsum("qkgd,nkd->kgqn", q[a:a + nq].view(nq, kv, h // kv, d), k[b:b + nk])
        if s["query_splits"] is not None:
          x = x.masked_fill(torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1), -math.inf)
        own_score[c] = (a, b, x.reshape(h, nq, nk))
      a, b = a + nq, b + nk
  lse = torch.zeros(q.shape[0], h, dtype=torch.float64, device="cuda")
  for i in range(h):
    j = i // (h // kv)
    for at in range(0, q.shape[0], 1024):
      score = q[at:at + 1024, i] @ s["prefix_key"][:, j].double().t()
      lse[at:at + 1024, i] = torch.logsumexp(score, 1)
      out[at:at + 1024, i] = torch.softmax(score, 1) @ s["prefix_value"][:, j].double()
  for a, b, x in own_score.values():
    nq, nk = x.shape[1:]
    was = lse[a:a + nq].t()
    now = torch.logaddexp(was, torch.logsumexp(x, 2))
    p = torch.exp(x - now[..., None]).view(kv, h // kv, nq, nk)
    out[a:a + nq] = out[a:a + nq] * torch.exp(was - now).t()[..., None] + torch.einsum(
        "kgqn,nkd->qkgd", p, v[b:b + nk]).reshape(nq, h, d)
  return {"out": out}


def _exact_ce(s):
  """In pieces of the rows, so that 64-bit logits of a million candidates fit."""
  q, w = s["query"].double(), s["rows"].double()
  n, grad = q.shape[0], s["case"]["grad"]
  bias = 0.0 if s["bias"] is None else s["bias"].double()
  loss = torch.zeros(n, dtype=torch.float64, device="cuda")
  dq, dw = torch.zeros_like(q), torch.zeros_like(w)
  db = torch.zeros(w.shape[0], dtype=torch.float64, device="cuda")
  step = max(1, 2 ** 29 // w.shape[0])
  for at in range(0, n, step):
    x = q[at:at + step] @ w.t() + bias
    lab = s["labels"][at:at + step]
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    has = (lab >= 0).double()
    loss[at:at + step] = -logp.gather(1, lab.clamp(min=0)[:, None])[:, 0] * has
    if grad:
      g = s["weight"][at:at + step].double() * has
      p = logp.exp_()
      p.scatter_add_(1, lab.clamp(min=0)[:, None], torch.full_like(g, -1.0)[:, None])
      p *= g[:, None]
      dq[at:at + step] = p @ w
      dw += p.t() @ q[at:at + step]
      db += p.sum(0)
  res = {"loss": loss}
  if grad:
    res.update(dquery=dq, drows=dw)
    if s["bias"] is not None:
      res["dbias"] = db
  return res
