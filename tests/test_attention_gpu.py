"""GPU: ragged attention (forward, gradient), the shared prefix form and the Attention combiner against
64-bit restatements with a bound per element (tests/seq_ref.py)."""
import numpy as np
import pytest
import torch

from tests import seq_ref

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def dev():
  return torch.device("cuda", 0)


def rows(rng, shape, dtype, scale=1.0):
  """(GPU tensor, the same values in 64 bits)."""
  t = torch.from_numpy(rng.standard_normal(shape) * scale).to(TYPES[dtype])
  return t.to(dev()), t.double().numpy()


def splits(lens, first=0):
  return np.concatenate([[first], first + np.cumsum(lens)]).astype(np.int64)


def on(x):
  return torch.from_numpy(x).to(dev())


def run_both(rng, dtype, H, Hkv, D, lq, lk, causal=False, mask=None, shared=False, scale=None, grad=True,
             pad=(0, 0)):
  """Random rows of the given lengths (lq None: one query each) through operator and restatement."""
  from monolith_amd import attention_ops
  ks = splits(lk, pad[0])
  qs = None if lq is None else splits(lq, pad[0])
  nq = len(lk) if lq is None else int(qs[-1]) + pad[1]
  nk = int(ks[-1]) + pad[1]
  q, q64 = rows(rng, (nq, H, D), dtype)
  k, k64 = rows(rng, (nk, Hkv, D), dtype)
  v, v64 = (None, k64) if shared else rows(rng, (nk, Hkv, D), dtype)
  g, g64 = rows(rng, (nq, H, D), dtype)
  m = None if mask is None else rng.random(nk) >= mask
  if grad:
    for t in (q, k, v):
      if t is not None:
        t.requires_grad_()
  got = attention_ops.ragged_attention(q, k, v, on(ks), None if qs is None else on(qs),
                                       None if m is None else on(m), causal, scale)
  segs = seq_ref.segments(qs, ks)
  want = seq_ref.attention(q64, k64, v64, segs, seq_ref.keep_rule(segs, m, causal),
                           D ** -0.5 if scale is None else scale, dtype, g64 if grad else None)
  seq_ref.check(got, want["out"], "out")
  if grad:
    got.backward(g)
    seq_ref.check(q.grad, want["dq"], "dq")
    seq_ref.check(k.grad, want["dkv" if shared else "dk"], "dk")
    if not shared:
      seq_ref.check(v.grad, want["dv"], "dv")


EDGES = [0, 1, 2, 15, 16, 17, 31, 0, 33, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 16), (4, 2, 32), (3, 1, 64), (2, 2, 128)])
@pytest.mark.parametrize("causal,mask", [(False, None), (True, None), (True, 0.3), (False, 0.9)])
def test_self_attention(dtype, H, Hkv, D, causal, mask):
  rng = np.random.default_rng(hash((D, causal)) % 1000)
  run_both(rng, dtype, H, Hkv, D, EDGES, EDGES, causal, mask)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [1, 3, 8, 12, 24, 40, 72, 100, 127])
def test_odd_dims(dtype, D):
  rng = np.random.default_rng(D)
  run_both(rng, dtype, 2, 1, D, [5, 70, 1], [9, 70, 33], D % 2 == 0, 0.2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 8), (1, 1, 16), (1, 1, 32), (2, 2, 64), (4, 1, 16), (8, 2, 64),
                                     (12, 1, 32), (40, 1, 16), (2, 1, 128), (1, 1, 5), (6, 2, 20)])
@pytest.mark.parametrize("shared,mask", [(True, 0.4), (False, None), (True, None), (False, 0.4)])
def test_one_query_per_row(dtype, H, Hkv, D, shared, mask):
  rng = np.random.default_rng(7 * H + D)
  run_both(rng, dtype, H, Hkv, D, None, [3, 0, 1, 64, 65, 300, 7, 31, 32, 33], mask=mask, shared=shared)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 32), (4, 2, 64), (16, 1, 16)])
def test_long_histories_are_split(dtype, H, Hkv, D):
  rng = np.random.default_rng(H)
  run_both(rng, dtype, H, Hkv, D, None, [20011, 5, 0, 1030], mask=0.1, shared=True)
  run_both(rng, dtype, H, Hkv, D, [2, 3, 1, 4], [9011, 5, 0, 1030], causal=True)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_one_long_history_among_short_ones(dtype):
  """Parts of equal keys: most sequences have one, some none, one has hundreds."""
  rng = np.random.default_rng(30)
  lens = [1, 0, 0, 700, 2, 150000, 0, 129, 1, 0]
  run_both(rng, dtype, 2, 1, 16, None, lens, mask=0.2, pad=(3, 70))
  run_both(rng, dtype, 3, 1, 8, None, lens, shared=True)
  run_both(rng, dtype, 5, 1, 8, None, [1, 0, 9000, 3])
  # the card full of short sequences, and some that are cut; batches around one part
  many = list(rng.integers(0, 4, 4500)) + [2048, 2049, 0, 4096, 4097, 9001] + list(rng.integers(0, 3, 300))
  run_both(rng, dtype, 1, 1, 4, None, many, mask=0.1)
  for lens in ([1024], [1025], [1023, 0, 1], [600, 600], [1024, 1, 1024], [0, 2049, 2560, 3], [127, 385]):
    run_both(rng, dtype, 2, 2, 8, None, lens, shared=True)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_few_keys_under_many_queries(dtype):
  """The pass over keys splits the queries: the keys' gradients are joined from partial sums."""
  rng = np.random.default_rng(3)
  run_both(rng, dtype, 4, 2, 32, [5000, 1, 900], [20, 3, 100])
  run_both(rng, dtype, 2, 2, 32, [3000], [3000], causal=True)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_cross_lengths_and_causal_alignment(dtype):
  """More keys than queries (a decoding step behind a cache) and fewer (the first queries see none)."""
  rng = np.random.default_rng(4)
  run_both(rng, dtype, 2, 1, 32, [1, 7, 70, 10, 4], [40, 100, 71, 3, 0], causal=True)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_sharp_and_flat_softmax(dtype):
  rng = np.random.default_rng(5)
  run_both(rng, dtype, 2, 2, 16, [50, 90], [50, 90], scale=6.0, causal=True)
  run_both(rng, dtype, 2, 2, 16, None, [50, 90], scale=6.0)
  run_both(rng, dtype, 2, 2, 16, [50, 90], [50, 90], scale=1e-6)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lq", [None, [40, 3, 100]])
def test_rows_of_no_sequence(dtype, lq):
  """A padded buffer: rows in front of the first split and behind the last hold anything and get zeros."""
  from monolith_amd import attention_ops
  rng = np.random.default_rng(6)
  lk = [40, 3, 100]
  ks, qs = splits(lk, 5), None if lq is None else splits(lq, 5)
  nk, nq = 5 + 143 + 77, 3 if lq is None else 5 + 143 + 77
  k, _ = rows(rng, (nk, 2, 32), dtype)
  q, _ = rows(rng, (nq, 2, 32), dtype)
  v, _ = rows(rng, (nk, 2, 32), dtype)
  for t in (k, v) if lq is None else (q, k, v):
    t[:5], t[148:] = float("nan"), float("inf")
  for t in (q, k, v):
    t.requires_grad_()
  out = attention_ops.ragged_attention(q, k, v, on(ks), None if qs is None else on(qs))
  g = torch.ones_like(out)
  dq, dk, dv = torch.autograd.grad(out, (q, k, v), g)
  # (the tiles are cut by the rows per sequence of the whole buffer, so a call without the padding may
  # sum in another order: the restatement says what the rows inside have to be)
  wide = lambda t: t.detach().double().cpu().numpy()
  segs = seq_ref.segments(qs, ks)
  want = seq_ref.attention(wide(q), wide(k), wide(v), segs, seq_ref.keep_rule(segs, None, False),
                           32 ** -0.5, dtype, wide(g))
  for got, name in ((out, "out"), (dq, "dq"), (dk, "dk"), (dv, "dv")):
    seq_ref.check(got, want[name], name)
  for t in (dk, dv) if lq is None else (out, dq, dk, dv):
    assert (t[:5] == 0).all() and (t[148:] == 0).all()
    assert torch.isfinite(t.float()).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("one", [True, False])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), torch.finfo(torch.float32).min])
def test_masked_places_hold_anything(dtype, one, bad):
  from monolith_amd import attention_ops
  rng = np.random.default_rng(8)
  lens = [30, 4, 90]
  s = on(splits(lens))
  k, _ = rows(rng, (124, 2, 16), dtype)
  v, _ = rows(rng, (124, 2, 16), dtype)
  q, _ = rows(rng, (3 if one else 124, 4, 16), dtype)
  mask = torch.from_numpy(rng.random(124) > 0.4).to(dev())
  mask[30:34] = False  # a sequence that nobody sees
  k2, v2 = k.clone(), v.clone()
  k2[~mask], v2[~mask] = bad, bad
  res = []
  for kk, vv in ((k, v), (k2, v2)):
    leaves = [t.clone().requires_grad_() for t in (q, kk, vv)]
    out = attention_ops.ragged_attention(*leaves, s, None if one else s, mask)
    res.append([out.detach()] + list(torch.autograd.grad(out, leaves, torch.ones_like(out))))
  for a, b in zip(*res):
    assert torch.isfinite(a.float()).all() and torch.equal(a, b)
  empty = slice(1, 2) if one else slice(30, 34)
  assert (res[0][0][empty] == 0).all() and (res[0][1][empty] == 0).all()
  assert (res[0][2][~mask] == 0).all() and (res[0][3][~mask] == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("one", [True, False])
def test_strides_and_alignment(dtype, one):
  """Packed projections, transposed heads, expanded rows and addresses off the 16-byte grid."""
  from monolith_amd import attention_ops
  rng = np.random.default_rng(9)
  n, H, D = 130, 4, 32
  s = on(splits([50, 80]))
  packed, _ = rows(rng, (n, 3, H, D), dtype)
  turned, _ = rows(rng, (H, n, D), dtype)
  odd, _ = rows(rng, (n * H * D + 1,), dtype)
  wide, _ = rows(rng, (n, H, D, 2), dtype)
  single, _ = rows(rng, (n, 1, D), dtype)
  forms = [packed[:, 1], turned.transpose(0, 1), odd[1:].view(n, H, D), wide[..., 1],
           single.expand(n, H, D)]
  for x in forms:
    q = (x[:2] if one else x).detach()
    args = (s, None if one else s)
    res = []
    for t in (x, x.contiguous()):
      leaves = [q if t is x else q.contiguous(), t, t]
      leaves = [y.detach().requires_grad_() for y in leaves]
      out = attention_ops.ragged_attention(*leaves, *args)
      g = torch.ones((), dtype=out.dtype, device=out.device).expand_as(out)
      res.append([out.detach()] + list(torch.autograd.grad(out, leaves, g)))
    for a, b in zip(*res):
      assert torch.equal(a, b)


def test_two_dimensional_rows_are_one_head():
  from monolith_amd import attention_ops
  rng = np.random.default_rng(10)
  k, _ = rows(rng, (40, 24), "fp32")
  q, _ = rows(rng, (2, 24), "fp32")
  s = on(splits([13, 27]))
  k.requires_grad_()
  out = attention_ops.ragged_attention(q, k, None, s)
  assert out.shape == (2, 24)
  want = attention_ops.ragged_attention(q.unsqueeze(1), k.unsqueeze(1), None, s)
  assert torch.equal(out, want[:, 0])
  out.sum().backward()
  assert k.grad.shape == k.shape


@pytest.mark.parametrize("nq,B,nk", [(0, 0, 0), (0, 3, 0), (3, 3, 0), (0, 1, 7), (0, 0, 2000)])
def test_nothing_to_do(nq, B, nk):
  from monolith_amd import attention_ops
  q = torch.randn(nq, 2, 16, device=dev(), requires_grad=True)
  k = torch.randn(nk, 1, 16, device=dev(), requires_grad=True)
  ks = torch.zeros(B + 1, dtype=torch.int64, device=dev())
  ks[-1] = nk if B else 0
  qs = torch.zeros_like(ks)
  qs[-1] = nq
  out = attention_ops.ragged_attention(q, k, None, ks, qs)
  assert out.shape == q.shape and (out == 0).all()
  dq, dk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
  assert (dq == 0).all() and dk.shape == k.shape and (dk == 0).all()


def test_gradient_against_differences():
  """|gradient| against the loss at x + h u and x - h u along the gradient, |u| = 1, h = 2^-5, in 32 bits
  through the operator. Off by h^2 / 6 = 1.7e-4 times the third derivative along u: a query's logits
  move by at most 0.25 |u_i| |k| <= 1.5 |u_i|, its output by at most 6 * 1.5^3 |u_i|^3 |g| |v| with
  |g| |v| <= 20, and the |u_i|^3 add up to 1 at most: under 0.07. Rounding is 2^-24 |loss| / h, far less."""
  from monolith_amd import attention_ops
  rng = np.random.default_rng(11)
  s = on(splits([40, 90, 3]))
  for one in (True, False):
    q, _ = rows(rng, (3 if one else 133, 2, 16), "fp32")
    k, _ = rows(rng, (133, 1, 16), "fp32")
    v, _ = rows(rng, (133, 1, 16), "fp32")
    g = torch.from_numpy(rng.standard_normal(tuple(q.shape))).to(dev())

    def loss(*x):
      return (attention_ops.ragged_attention(*x, s, None if one else s).double() * g).sum()

    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i in range(3):
      x = [q, k, v]
      size = grads[i].double().norm().item()
      u = (grads[i].double() / size).float()
      up, down = list(x), list(x)
      up[i], down[i] = x[i] + 2.0 ** -5 * u, x[i] - 2.0 ** -5 * u
      with torch.no_grad():
        diff = ((loss(*up) - loss(*down)) * 16).item()
      assert abs(diff - size) <= 0.07, (one, i, diff, size)


def capture(fn, replays, between):
  """Record fn() once on a side stream after a warm-up and replay it."""
  st = torch.cuda.Stream()
  st.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(st):
    fn()
  torch.cuda.current_stream().wait_stream(st)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = fn()
  for i in range(replays):
    between(i)
    graph.replay()
    yield out


@pytest.mark.parametrize("lens", [[30, 70, 200], [4000, 9, 100]])
@pytest.mark.parametrize("one", [True, False])
def test_captured_forward_and_backward(lens, one):
  """A training step in a graph, replayed on other inputs and other lengths with eager work between."""
  from monolith_amd import attention_ops
  rng = np.random.default_rng(12)
  n = sum(lens)
  nq = 3 if one else n
  mk = lambda m: torch.from_numpy(rng.standard_normal((m, 2, 32))).to(dev(), torch.float32)
  q, k, v, g = mk(nq), mk(n), mk(n), mk(nq)
  s = on(splits(lens))

  def step(q, k, v):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention_ops.ragged_attention(*leaves, s, None if one else s, causal=not one)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, g))

  eager = []

  def between(i):
    lens2 = lens if i == 0 else list(rng.permutation(lens))
    s.copy_(on(splits(lens2)))
    for t in (q, k, v, g):
      t.copy_(mk(t.shape[0]))
    eager[:] = [x.clone() for x in step(q, k, v)]
    torch.cuda.synchronize()

  for got in capture(lambda: step(q, k, v), 4, between):
    torch.cuda.synchronize()
    for a, b in zip(got, eager):
      assert torch.equal(a, b)


def test_results_do_not_change_from_call_to_call_or_stream():
  from monolith_amd import attention_ops
  rng = np.random.default_rng(13)
  lens = [700, 33, 1200]
  s = on(splits(lens))
  for dtype in ("fp32", "bf16"):
    for one in (True, False):
      q, _ = rows(rng, (3 if one else sum(lens), 4, 32), dtype)
      k, _ = rows(rng, (sum(lens), 2, 32), dtype)

      def step():
        leaves = [t.detach().requires_grad_() for t in (q, k)]
        out = attention_ops.ragged_attention(*leaves, None, s, None if one else s)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, torch.ones_like(out)))

      first = step()
      side = [torch.cuda.Stream(), torch.cuda.Stream()]
      runs = []
      for st in side:  # two calls at once, each on a stream and a workspace of its own
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
          runs.append(step())
      torch.cuda.synchronize()
      for r in runs + [step()]:
        for a, b in zip(first, r):
          assert torch.equal(a, b)


def test_query_gradient_alone():
  from monolith_amd import attention_ops
  rng = np.random.default_rng(14)
  s = on(splits([20, 30]))
  for qs in (None, s):
    q, _ = rows(rng, (2 if qs is None else 50, 2, 16), "fp32")
    k, _ = rows(rng, (50, 2, 16), "fp32")
    full = [t.clone().requires_grad_() for t in (q, k)]
    want = torch.autograd.grad(attention_ops.ragged_attention(*full, None, s, qs).sum(), full[0])[0]
    alone = q.clone().requires_grad_()
    attention_ops.ragged_attention(alone, k, None, s, qs).sum().backward()
    assert torch.equal(alone.grad, want)


# ---- the shared prefix ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 16), (4, 2, 32), (8, 1, 64), (2, 2, 128), (3, 3, 10)])
@pytest.mark.parametrize("prefix,lq,lk", [
    (1, None, [0, 1, 3]), (300, None, None), (300, None, [0, 40, 7, 64, 1]), (0, None, [4, 0, 9]),
    (77, [1, 3, 2, 0, 70], [5, 3, 40, 6, 70]), (5000, [1, 2], [0, 2]), (5000, [3, 1, 2], None),
    (2000, [50] * 6, [60] * 6), (40, None, [3000, 5, 0, 700]), (40, [2, 1, 3], [3000, 5, 700])])
def test_shared_prefix(dtype, H, Hkv, D, prefix, lq, lk):
  """Every query over the prefix and its own keys: the restatement has both as one list of keys."""
  from monolith_amd import attention_ops
  rng = np.random.default_rng(prefix + H)
  B = len(lk) if lk is not None else 5 if lq is None else len(lq)
  lens = lq if lq is not None else [1] * B
  q, q64 = rows(rng, (sum(lens), H, D), dtype)
  pk, pk64 = rows(rng, (prefix, Hkv, D), dtype)
  pv, pv64 = rows(rng, (prefix, Hkv, D), dtype)
  nk = sum(lk) if lk is not None else 0
  k, k64 = rows(rng, (nk, Hkv, D), dtype)
  v, v64 = rows(rng, (nk, Hkv, D), dtype)
  pm, km = rng.random(prefix) > 0.1, rng.random(nk) > 0.1
  causal = lq is not None and lk is not None
  kw = dict(prefix_mask=on(pm), causal=causal)
  if lk is not None:
    kw.update(key=k, value=v, key_splits=on(splits(lk)), key_mask=on(km))
  if lq is not None:
    kw["query_splits"] = on(splits(lq))
  got = attention_ops.shared_prefix_attention(q, pk, pv, **kw)
  qs, ks = splits(lens), splits(lk if lk is not None else [0] * B)
  segs = [(np.arange(qs[b], qs[b + 1]), np.concatenate([np.arange(prefix), prefix + np.arange(ks[b], ks[b + 1])]))
          for b in range(B)]
  mask = np.concatenate([pm, km])

  def keep(c, n, m):
    ok = np.ones((n, m), bool)
    if causal:
      own = m - prefix
      ok[:, prefix:] = np.arange(own)[None] <= np.arange(n)[:, None] + own - n
    return ok & mask[segs[c][1]][None]

  want = seq_ref.attention(q64, np.concatenate([pk64, k64]), np.concatenate([pv64, v64]), segs, keep,
                           D ** -0.5, dtype)
  # the two parts are joined in 32 bits: one more exponential, product and sum for every part
  value, bound = want["out"]
  seq_ref.check(got, (value, bound * (1 + 2.0 ** -10) + 64 * seq_ref.U32 * np.abs(value)), "out")


def test_shared_prefix_captured_and_repeated():
  from monolith_amd import attention_ops
  rng = np.random.default_rng(15)
  q, _ = rows(rng, (9, 4, 32), "bf16")
  pk, _ = rows(rng, (3000, 2, 32), "bf16")
  k, _ = rows(rng, (30, 2, 32), "bf16")
  s = on(splits([4, 0, 6, 1, 2, 3, 5, 7, 2]))
  eager = []

  def between(i):
    q.copy_(rows(rng, (9, 4, 32), "bf16")[0])
    pk.copy_(rows(rng, (3000, 2, 32), "bf16")[0])
    eager[:] = [attention_ops.shared_prefix_attention(q, pk, None, k, None, s)]

  for got in capture(lambda: attention_ops.shared_prefix_attention(q, pk, None, k, None, s), 3, between):
    torch.cuda.synchronize()
    assert torch.equal(got, eager[0])
