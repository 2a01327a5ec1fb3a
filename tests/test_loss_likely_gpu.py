"""GPU: softmax cross entropy where the label is the likely candidate, as it is once a model has learned:
loss and gradient come from 1 - p of the label, which is small, and have to keep their digits."""
import numpy as np
import pytest
import torch

from tests.seq_ref import HALF, U32, check
from tests.test_attention_gpu import TYPES, dev, on

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def exact(q, w, labels, bias, scale, g):
  """(loss, dquery, drows, dbias), |p - hot|, the label's probability and the largest magnitude that a query's
  logits sum up, in 64 bits."""
  n = len(q)
  l = scale * (q @ w.T) + (0 if bias is None else bias)
  S = (scale * np.abs(q) @ np.abs(w).T + (0 if bias is None else np.abs(bias))).max(1)
  hit = l[np.arange(n), labels]
  others = np.exp(l - hit[:, None])  # relative to the label's own
  others[np.arange(n), labels] = 0
  z = others.sum(1)
  p = others / (1 + z)[:, None]
  d = p.copy()  # p - hot
  d[np.arange(n), labels] = -z / (1 + z)
  ds = d * g[:, None]
  return (np.log1p(z), scale * ds @ w, scale * ds.T @ q, ds.sum(0)), np.abs(d), 1 / (1 + z), S


def weights_error(S, D, V):
  """Of a weight p relative to it: a logit is D products and sums and two roundings of S, those of fp32 rows
  drop up to two more of a product, its base change and the subtraction of the log-sum (at most S + log V)
  two each, the exponential two, the sum of V terms one each."""
  return 2 * U32 * ((D + 4) * S + 4 * 1.4427 * (S + np.log(V) + 1) + 4) + 2 * U32 * (V + 8)


def run(q, w, labels, bias, scale, g):
  from monolith_amd import loss_ops
  leaves = [t.detach().requires_grad_() for t in (q, w)] + ([] if bias is None else [bias.detach().requires_grad_()])
  loss = loss_ops.softmax_cross_entropy(leaves[0], leaves[1], on(labels), None if bias is None else leaves[2], scale)
  return [loss.detach()] + list(torch.autograd.grad(loss, leaves, g))


def aligned(rng, dtype, n, V, D, lo, hi):
  """Queries along their label's row, lo .. hi times as long."""
  w = torch.from_numpy(rng.standard_normal((V, D)) * 2 / D ** 0.5).to(TYPES[dtype])
  labels = rng.integers(0, V, n)
  c = rng.uniform(lo, hi, (n, 1))
  q = torch.from_numpy(w.double().numpy()[labels] * c + 0.1 * rng.standard_normal((n, D))).to(TYPES[dtype])
  return q, w, labels


# one piece of candidates and several; queries in tiles of one and two columns a wave
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,V,D", [(500, 60, 64), (300, 1000, 64), (700, 1500, 32), (200, 3000, 128), (90, 700, 256)])
@pytest.mark.parametrize("bias", [False, True])
def test_gradients_of_likely_labels(dtype, n, V, D, bias):
  """Every weight, the label's p - 1 among them, is rounded to the type once; sums are 32 bits."""
  rng = np.random.default_rng(V + D)
  q, w, labels = aligned(rng, dtype, n, V, D, 1.5, 5.0)
  b = rng.uniform(0, 1, V).astype(np.float32) if bias else None
  g = rng.uniform(0.5, 1.5, n).astype(np.float32)
  q64, w64, g64 = q.double().numpy(), w.double().numpy(), g.astype(np.float64)
  want, d, p, S = exact(q64, w64, labels, None if b is None else b.astype(np.float64), 1.0, g64)
  assert p.min() < 0.95 and np.quantile(p, 0.8) > 0.99
  got = run(q.to(dev()), w.to(dev()), labels, None if b is None else on(b), 1.0, on(g))
  half, e = HALF[dtype], weights_error(S, D, V)[:, None]
  hot = np.zeros_like(d)
  hot[np.arange(n), labels] = 1
  off = np.abs(g64)[:, None] * ((half + (V + n + 4) * U32) * d + (e + 4 * U32) * np.where(hot, p[:, None], d) +
                                4 * U32 * hot)
  oq, ow = off @ np.abs(w64), off.T @ np.abs(q64)
  check(got[1], (want[1], oq + half * (np.abs(want[1]) + oq)), "dquery")
  check(got[2], (want[2], ow + half * (np.abs(want[2]) + ow)), "drows")
  if bias:
    check(got[3], (want[3], off.sum(0) + U32 * np.abs(want[3])), "dbias")


@pytest.mark.parametrize("n,V,D", [(500, 60, 64), (300, 1000, 64), (700, 1500, 32), (200, 3000, 128), (90, 700, 256)])
def test_rows_of_the_query_gradient(n, V, D):
  """Nine of ten bf16 rows are off by less than two roundings to the type in all: a row's error is that of its
  weights, independent of each other and at most half a step each, and its own rounding."""
  rng = np.random.default_rng(V + D)
  q, w, labels = aligned(rng, "bf16", n, V, D, 1.5, 5.0)
  want = exact(q.double().numpy(), w.double().numpy(), labels, None, 1.0, np.ones(n))[0][1]
  got = run(q.to(dev()), w.to(dev()), labels, None, 1.0, torch.ones(n, device=dev()))[1].double().cpu().numpy()
  off = np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)
  assert np.quantile(off, 0.9) <= 2 * HALF["bf16"], np.quantile(off, [0.1, 0.5, 0.9])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,pairs,D,scale", [(40, 4, 16, 1.0), (300, 64, 32, 20.0), (300, 900, 64, 0.05)])
@pytest.mark.parametrize("bias", [False, True])
def test_digits_of_a_sharp_loss(dtype, n, pairs, D, scale, bias):
  """Logits of about 100 and a second candidate much like the label, 2 to 9 below it: loss and gradients are 1 - p,
  from 1e-1 to 1e-4, times what one 32-bit sum leaves, not the difference of numbers of size 100."""
  rng = np.random.default_rng(pairs)
  first = rng.standard_normal((pairs, D)) / D ** 0.5
  w = torch.from_numpy(np.concatenate([first, first * (1 - rng.uniform(0.02, 0.09, (pairs, 1)))])).to(TYPES[dtype])
  labels = rng.integers(0, pairs, n)
  w64 = w.double().numpy()
  q = torch.from_numpy(w64[labels] * 100 / (w64[labels] ** 2).sum(1, keepdims=True) / scale).to(TYPES[dtype])
  b = rng.uniform(-1, 1, 2 * pairs).astype(np.float32) if bias else None
  g = rng.uniform(0.5, 1.5, n).astype(np.float32)
  q64, g64 = q.double().numpy(), g.astype(np.float64)
  want, d, p, S = exact(q64, w64, labels, None if b is None else b.astype(np.float64), scale, g64)
  assert 1e-5 < np.median(1 - p) < 0.2
  got = run(q.to(dev()), w.to(dev()), labels, None if b is None else on(b), scale, on(g))
  half, e = HALF[dtype], weights_error(S, D, 2 * pairs)
  # the loss is the sum of the others' weights relative to the label's, its logarithm's argument and value round
  check(got[0], (want[0], e * want[0] + 8 * U32 * want[0]), "loss")
  assert (got[0] >= 0).all()
  off = np.abs(g64)[:, None] * (half + e[:, None] + (2 * pairs + n + 8) * U32) * d
  oq, ow = scale * off @ np.abs(w64), scale * off.T @ np.abs(q64)
  check(got[1], (want[1], oq + half * (np.abs(want[1]) + oq)), "dquery")
  check(got[2], (want[2], ow + half * (np.abs(want[2]) + ow)), "drows")
  if bias:
    check(got[3], (want[3], off.sum(0) + U32 * np.abs(want[3])), "dbias")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("V", [1, 200])
def test_no_other_candidate(dtype, sign, V):
  """The label is the only candidate, with a logit far from 0: no loss and no gradient."""
  rng = np.random.default_rng(5)
  w = torch.from_numpy(rng.standard_normal((V, 16))).to(TYPES[dtype])
  q = (sign * 30 * w[:1]).expand(40, 16)
  bias = None
  if V > 1:
    bias = torch.full((V,), -float("inf"), device=dev())
    bias[0] = 0
  for t in run(q.to(dev()), w.to(dev()), np.zeros(40, np.int64), bias, 1.0, torch.ones(40, device=dev())):
    assert (t == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_labels_far_from_likely(dtype):
  """1 - p is 1 as far as 32 bits go, and the loss the distance to the others, up to hundreds."""
  rng = np.random.default_rng(6)
  q, w, labels = aligned(rng, dtype, 200, 300, 32, -40.0, 5.0)
  g = rng.uniform(0.5, 1.5, 200).astype(np.float32)
  q64, w64, g64 = q.double().numpy(), w.double().numpy(), g.astype(np.float64)
  want, d, p, S = exact(q64, w64, labels, None, 1.0, g64)
  assert want[0].max() > 100 and want[0].min() < 1
  got = run(q.to(dev()), w.to(dev()), labels, None, 1.0, on(g))
  half, e = HALF[dtype], weights_error(S, 32, 300)
  check(got[0], (want[0], e * (1 - p) + 8 * U32 * want[0]), "loss")
  off = np.abs(g64)[:, None] * (half + e[:, None] + 508 * U32) * d
  oq, ow = off @ np.abs(w64), off.T @ np.abs(q64)
  check(got[1], (want[1], oq + half * (np.abs(want[1]) + oq)), "dquery")
  check(got[2], (want[2], ow + half * (np.abs(want[2]) + ow)), "drows")
