"""GPU: softmax cross entropy against embedding rows and its gradient, against a 64-bit restatement with
a bound per element (tests/seq_ref.py), and together with the table whose rows it trains."""
import numpy as np
import pytest
import torch

from tests import seq_ref
from tests.test_attention_gpu import capture, dev, on, rows

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def run_both(rng, dtype, n, V, D, bias=True, scale=1.0, special=True):
  from monolith_amd import loss_ops
  q, q64 = rows(rng, (n, D), dtype)
  w, w64 = rows(rng, (V, D), dtype, 2.0 / D ** 0.5)
  labels = rng.integers(0, V, n)
  b64 = None
  if bias:
    b = rng.standard_normal(V).astype(np.float32)
    if special and V > 4:
      b[rng.random(V) < 0.2] = -np.inf
    b64 = b.astype(np.float64)
  if special and n > 6:
    labels[0], labels[1], labels[2], labels[3] = -1, V, -2, 2 ** 40
  g64 = rng.standard_normal(n)
  g = on(g64.astype(np.float32))
  g64 = g.double().cpu().numpy()
  q.requires_grad_()
  w.requires_grad_()
  bt = None if b64 is None else on(b).requires_grad_()
  loss = loss_ops.softmax_cross_entropy(q, w, on(labels), bt, scale)
  want = seq_ref.cross_entropy(q64, w64, labels, b64, scale, dtype, g64)
  assert loss.dtype == torch.float32
  seq_ref.check(loss, want["loss"], "loss")
  loss.backward(g)
  seq_ref.check(q.grad, want["dq"], "dquery")
  seq_ref.check(w.grad, want["dw"], "drows")
  if bt is not None:
    seq_ref.check(bt.grad, want["db"], "dbias")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [1, 7, 8, 16, 20, 32, 48, 64, 100, 128, 192, 250, 256])
def test_dims(dtype, D):
  rng = np.random.default_rng(D)
  run_both(rng, dtype, 150, 333, D, bias=D % 3 != 0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n,V", [(1, 1), (1, 2), (3, 1), (1, 5000), (2000, 3), (64, 64), (127, 129), (129, 65),
                                 (700, 2000), (33, 20011)])
@pytest.mark.parametrize("bias", [True, False])
def test_sizes(dtype, n, V, bias):
  rng = np.random.default_rng(n + V)
  run_both(rng, dtype, n, V, 32, bias)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_temperature(dtype):
  rng = np.random.default_rng(1)
  run_both(rng, dtype, 100, 500, 16, True, 8.0)
  run_both(rng, dtype, 100, 500, 16, False, 0.01)


def test_no_queries():
  from monolith_amd import loss_ops
  q = torch.zeros(0, 16, device=dev(), requires_grad=True)
  w = torch.randn(40, 16, device=dev(), requires_grad=True)
  b = torch.randn(40, device=dev(), requires_grad=True)
  loss = loss_ops.softmax_cross_entropy(q, w, torch.zeros(0, dtype=torch.int64, device=dev()), b)
  dq, dw, db = torch.autograd.grad(loss, (q, w, b), torch.zeros_like(loss))
  assert loss.shape == (0,) and dq.shape == q.shape and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_excluded_candidates_hold_anything(dtype, bad):
  """A candidate with a bias of -inf, a query without a label: what they hold reaches nothing else."""
  from monolith_amd import loss_ops
  rng = np.random.default_rng(2)
  q, _ = rows(rng, (100, 32), dtype)
  w, _ = rows(rng, (300, 32), dtype)
  labels = torch.from_numpy(rng.integers(0, 100, 100)).to(dev())
  labels[5], labels[6] = -1, 250
  bias = torch.zeros(300, device=dev())
  bias[200:] = -float("inf")
  g = torch.randn(100, device=dev())
  g2 = g.clone()
  g2[5:7] = bad
  q2, w2 = q.clone(), w.clone()
  w2[200:] = bad
  q2[5:7] = bad
  res = []
  for a, b, gg in ((q, w, g), (q2, w2, g2)):
    leaves = [a.clone().requires_grad_(), b.clone().requires_grad_(), bias.clone().requires_grad_()]
    loss = loss_ops.softmax_cross_entropy(leaves[0], leaves[1], labels, leaves[2])
    res.append([loss.detach()] + list(torch.autograd.grad(loss, leaves, gg)))
  assert res[0][0][5] == 0 and res[0][0][6] == float("inf")
  for a, b in zip(*res):
    assert torch.equal(a, b)
  assert all(torch.isfinite(t.float()).all() for t in res[0][1:])
  assert (res[0][1][5:7] == 0).all() and (res[0][2][200:] == 0).all() and (res[0][3][200:] == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strides_and_alignment(dtype):
  from monolith_amd import loss_ops
  rng = np.random.default_rng(3)
  wide, _ = rows(rng, (200, 3, 32), dtype)
  odd, _ = rows(rng, (300 * 32 + 1,), dtype)
  turned, _ = rows(rng, (32, 300), dtype)
  labels = torch.from_numpy(rng.integers(0, 300, 200)).to(dev())
  one, _ = rows(rng, (1, 32), dtype)
  for q in (wide[:, 1], one.expand(200, 32)):
    for w in (odd[1:].view(300, 32), turned.t()):
      res = []
      for a, b in ((q, w), (q.contiguous(), w.contiguous())):
        leaves = [a.detach().requires_grad_(), b.detach().requires_grad_()]
        loss = loss_ops.softmax_cross_entropy(*leaves, labels)
        # (an expanded gradient: its stride is 0)
        res.append([loss.detach()] + list(torch.autograd.grad(loss.sum(), leaves)))
      for x, y in zip(*res):
        assert torch.equal(x, y)


def test_single_gradients_and_equal_results():
  from monolith_amd import loss_ops
  rng = np.random.default_rng(4)
  q, _ = rows(rng, (500, 32), "fp32")
  w, _ = rows(rng, (900, 32), "fp32")
  b = torch.randn(900, device=dev())
  labels = torch.from_numpy(rng.integers(0, 900, 500)).to(dev())
  full = [t.clone().requires_grad_() for t in (q, w, b)]
  want = torch.autograd.grad(loss_ops.softmax_cross_entropy(full[0], full[1], labels, full[2]).sum(), full)
  for i in range(3):
    x = [q, w, b]
    x[i] = x[i].clone().requires_grad_()
    got = torch.autograd.grad(loss_ops.softmax_cross_entropy(x[0], x[1], labels, x[2]).sum(), x[i])[0]
    assert torch.equal(got, want[i])


def test_captured_step():
  from monolith_amd import loss_ops
  rng = np.random.default_rng(5)
  q, _ = rows(rng, (300, 32), "fp32")
  w, _ = rows(rng, (1700, 32), "fp32")
  b = torch.randn(1700, device=dev())
  labels = torch.from_numpy(rng.integers(0, 1700, 300)).to(dev())
  g = torch.rand(300, device=dev())
  eager = []

  def step():
    leaves = [t.detach().requires_grad_() for t in (q, w, b)]
    loss = loss_ops.softmax_cross_entropy(leaves[0], leaves[1], labels, leaves[2])
    return [loss.detach()] + list(torch.autograd.grad(loss, leaves, g))

  def between(i):
    q.copy_(rows(rng, (300, 32), "fp32")[0])
    labels.copy_(torch.from_numpy(rng.integers(-1, 1700, 300)).to(dev()))
    eager[:] = [x.clone() for x in step()]
    torch.cuda.synchronize()

  for got in capture(step, 4, between):
    torch.cuda.synchronize()
    for x, y in zip(got, eager):
      assert torch.equal(x, y)


def test_gradient_against_differences():
  """|gradient| against the loss at x + h u and x - h u along the gradient, |u| = 1, h = 2^-5, in 32 bits
  through the operator. Off by h^2 / 6 = 1.7e-4 times the third derivative along u, a third cumulant of
  the logits' movement: at most 6 (|u_i| |w|)^3 for a query, |w| <= 3, and the |u_i|^3 add up to 1 at
  most: under 0.03 (a row's or a bias's share of one query is weighted by its probability, and u is
  spread over 400 of them). Rounding is 2^-24 |loss| / h, less than 1e-3."""
  from monolith_amd import loss_ops
  rng = np.random.default_rng(6)
  q, _ = rows(rng, (90, 16), "fp32")
  w, _ = rows(rng, (400, 16), "fp32", 0.5)
  b = torch.randn(400, device=dev())
  labels = torch.from_numpy(rng.integers(0, 400, 90)).to(dev())

  def loss(x):
    return loss_ops.softmax_cross_entropy(x[0], x[1], labels, x[2]).double().sum()

  leaves = [t.clone().requires_grad_() for t in (q, w, b)]
  grads = torch.autograd.grad(loss(leaves), leaves)
  for i in range(3):
    x = [q, w, b]
    size = grads[i].double().norm().item()
    u = (grads[i].double() / size).float()
    up, down = list(x), list(x)
    up[i], down[i] = x[i] + 2.0 ** -5 * u, x[i] - 2.0 ** -5 * u
    with torch.no_grad():
      diff = ((loss(up) - loss(down)) * 16).item()
    assert abs(diff - size) <= 0.03, (i, diff, size)
