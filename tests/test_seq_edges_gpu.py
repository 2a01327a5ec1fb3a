"""GPU: calls at the edges of what the sequence and loss operators allow."""
import numpy as np
import pytest
import torch

from tests import seq_ref
from tests.test_attention_gpu import dev, on, rows

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
