"""GPU: calls at the edges of what the sequence and loss operators allow."""
import numpy as np
import pytest
import torch

from tests import seq_ref
from tests.test_attention_gpu import dev, on, rows, splits

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
LOW = [-2e7, -1e10, -1e30, float(np.finfo(np.float32).min)]


def grads(out, leaves, g):
  return [out.detach()] + list(torch.autograd.grad(out, leaves, g))


# ---- masks by the lowest value -------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("scale", [1.0, 0.05, 20.0])
def test_biases_of_the_lowest_value(dtype, low, scale):
  """A run of candidates whose bias is as good as -inf has no weight, as with -inf: the same results. A label among
  them has the loss and the gradient of its definition."""
  from monolith_amd import loss_ops
  rng = np.random.default_rng(20)
  q, _ = rows(rng, (150, 32), dtype, scale ** -0.5)
  w, _ = rows(rng, (700, 32), dtype, scale ** -0.5)
  gone = torch.zeros(700, dtype=torch.bool)
  gone[:200] = gone[450:460] = gone[600:] = True
  gone = gone.to(dev())
  labels = on(rng.integers(200, 450, 150))
  g = torch.randn(150, device=dev())
  plain = torch.randn(700, device=dev())
  res = []
  for value in (-float("inf"), low):
    leaves = [q.clone().requires_grad_(), w.clone().requires_grad_(),
              torch.where(gone, value, plain).requires_grad_()]
    res.append(grads(loss_ops.softmax_cross_entropy(leaves[0], leaves[1], labels, leaves[2], scale), leaves, g))
  for a, b in zip(*res):
    assert torch.isfinite(a.float()).all() and torch.equal(a, b)
  labels[3] = 5  # the one label that is low
  leaves = [q.clone().requires_grad_(), w.clone().requires_grad_(), torch.where(gone, low, plain).requires_grad_()]
  loss, _, dw, db = grads(loss_ops.softmax_cross_entropy(leaves[0], leaves[1], labels, leaves[2], scale), leaves, g)
  # the rest of the loss is below 100, and each of its roundings one of 2e7 or more
  assert abs(loss[3].item() / -low - 1) <= 100 / 2e7 + 4 * seq_ref.U32
  assert torch.equal(db[5], -g[3])
  want = -g[3].double() * q[3].double() * scale
  half = seq_ref.HALF[dtype]
  assert ((dw[5].double() - want).abs() <= (2 * half + half * half + 4 * seq_ref.U32) * want.abs()).all()


# ---- queries without a key -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("form", ["causal", "mask", "one", "one_many_heads"])
def test_queries_without_a_key_hold_anything(dtype, bad, form):
  """Neither their rows nor what arrives as their gradient reaches a key's gradient."""
  from monolith_amd import attention_ops
  rng = np.random.default_rng(21)
  one = form.startswith("one")
  heads = 10 if form == "one_many_heads" else 4
  lk = [30, 40, 90, 5]
  lq = [1] * 4 if one else [100, 40, 130, 5]
  q, _ = rows(rng, (sum(lq), heads, 16), dtype)
  k, _ = rows(rng, (sum(lk), 2, 16), dtype)
  v, _ = rows(rng, (sum(lk), 2, 16), dtype)
  g, _ = rows(rng, (sum(lq), heads, 16), dtype)
  mask = torch.ones(sum(lk), dtype=torch.bool, device=dev())
  empty = np.zeros(sum(lq), bool)
  ks, qs = splits(lk), splits(lq)
  if form == "causal":
    for b in range(4):
      empty[qs[b]:qs[b] + max(0, lq[b] - lk[b])] = True
  else:
    mask[ks[1]:ks[2]] = False
    empty[qs[1]:qs[2]] = True
  assert empty.any()
  res = []
  for value in (0.0, bad):
    q2, g2 = q.clone(), g.clone()
    q2[on(empty)], g2[on(empty)] = value, value
    leaves = [t.clone().requires_grad_() for t in (q2, k, v)]
    out = attention_ops.ragged_attention(*leaves, on(ks), None if one else on(qs), None if form == "causal" else mask,
                                         form == "causal")
    res.append(grads(out, leaves, g2))
  for a, b in zip(*res):
    assert torch.isfinite(b.float()).all() and torch.equal(a, b)
  assert (res[1][0][on(empty)] == 0).all() and (res[1][1][on(empty)] == 0).all()


# ---- a padded request behind a prefix ------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("prefix", [1, 70, 5000])
@pytest.mark.parametrize("own", [None, [5, 0, 40, 3], [3000, 1, 2, 900]])
@pytest.mark.parametrize("heads", [2, 12])
def test_prefix_rows_of_no_sequence(dtype, prefix, own, heads):
  """Queries in front of the first split and behind the last hold anything and get zeros; the others get what
  they get without them."""
  from monolith_amd import attention_ops
  rng = np.random.default_rng(22)
  lq = [3, 70, 1, 20]
  qs = splits(lq, 37)
  nq = int(qs[-1]) + 150
  q, q64 = rows(rng, (nq, heads, 24), dtype)
  pk, pk64 = rows(rng, (prefix, 2, 24), dtype)
  pv, pv64 = rows(rng, (prefix, 2, 24), dtype)
  lk = own if own is not None else [0] * 4
  k, k64 = rows(rng, (sum(lk), 2, 24), dtype)
  v, v64 = rows(rng, (sum(lk), 2, 24), dtype)
  q[:37], q[int(qs[-1]):] = float("nan"), float("inf")
  kw = {} if own is None else dict(key=k, value=v, key_splits=on(splits(lk)), causal=True)
  out = attention_ops.shared_prefix_attention(q, pk, pv, query_splits=on(qs), **kw)
  assert (out[:37] == 0).all() and (out[int(qs[-1]):] == 0).all()
  ks = splits(lk)
  segs = [(np.arange(qs[b], qs[b + 1]), np.concatenate([np.arange(prefix), prefix + np.arange(ks[b], ks[b + 1])]))
          for b in range(4)]

  def keep(c, n, m):
    ok = np.ones((n, m), bool)
    ok[:, prefix:] = np.arange(m - prefix)[None] <= np.arange(n)[:, None] + m - prefix - n
    return ok

  want = seq_ref.attention(q64, np.concatenate([pk64, k64]), np.concatenate([pv64, v64]), segs, keep,
                           24 ** -0.5, dtype)["out"]
  live = slice(37, int(qs[-1]))
  # the parts are joined in 32 bits: one more exponential, product and sum for every part
  seq_ref.check(out[live], (want[0][live], (want[1] * (1 + 2.0 ** -10) + 64 * seq_ref.U32 * np.abs(want[0]))[live]),
                "out")


# ---- forward mode --------------------------------------------------------------------------------
def test_gradients_refuse_tangents():
  """A tangent that arrives with the output's gradient is refused as one in the inputs is."""
  from torch.autograd import forward_ad
  from monolith_amd import attention_ops, loss_ops
  q = torch.randn(4, 1, 16, device=dev(), requires_grad=True)
  k = torch.randn(9, 1, 16, device=dev())
  calls = (lambda: attention_ops.ragged_attention(q, k, None, on(np.array([0, 2, 4, 6, 9]))),
           lambda: loss_ops.softmax_cross_entropy(q[:, 0], k[:, 0], on(np.array([0, 3, 8, 1]))))
  for call in calls:
    with forward_ad.dual_level():
      out = call()
      weight = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
      with pytest.raises(ValueError, match="forward-mode"):
        torch.autograd.grad((out * weight).sum(), q)
      torch.autograd.grad(call().sum(), q)


# ---- numbers near the largest --------------------------------------------------------------------
def test_the_largest_finite_numbers():
  """fp32 rows near the largest number against keys near the smallest: products of ordinary size."""
  from monolith_amd import attention_ops, loss_ops
  rng = np.random.default_rng(23)
  big = float(np.finfo(np.float32).max)
  n, D = 40, 16
  x = np.sign(rng.standard_normal((n, D))) * big * (1 - rng.uniform(0, 2.0 ** -9, (n, D)))
  y = np.exp2(-125 - rng.integers(0, 2, (n, D))) * np.sign(rng.standard_normal((n, D)))  # (no bits behind the first)
  v, v64 = rows(rng, (n, 1, D), "fp32")
  x, y = (t.astype(np.float32) for t in (x, y))
  s = on(np.array([0, n]))
  out = attention_ops.ragged_attention(on(x).unsqueeze(1), on(y).unsqueeze(1), v, s, s, scale=0.25)
  x6, y6 = x.astype(np.float64), y.astype(np.float64)
  segs = seq_ref.segments(np.array([0, n]), np.array([0, n]))
  want = seq_ref.attention(x6[:, None], y6[:, None], v64, segs, seq_ref.keep_rule(segs, None, False), 0.25, "fp32")
  seq_ref.check(out, want["out"], "out")
  labels = rng.integers(0, n, n)
  for a, b in ((x, y), (y, x)):
    loss = loss_ops.softmax_cross_entropy(on(a), on(b), on(labels), None, 0.25)
    want = seq_ref.cross_entropy(a.astype(np.float64), b.astype(np.float64), labels, None, 0.25, "fp32")
    seq_ref.check(loss, want["loss"], "loss")
