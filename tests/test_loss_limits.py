"""The largest softmax cross entropies: what is refused (CPU) and what is not (GPU)."""
import ctypes as C

import pytest
import torch

from monolith_amd import _lib, loss_ops

MOST = 2 ** 31 - 2 ** 27


@pytest.mark.parametrize("which", ["grad_rows", "grad_bias"])
def test_gradients_of_too_many_rows_are_refused(which):
  """A launch of 2^32 threads would be none: refused before it, and before its workspace is made."""
  name = "mono_softmax_cross_entropy_gradient"
  for vocab, refused in ((MOST, True), (2 ** 31 - 70000, True), (MOST - 1, False)):
    a = _lib.SoftmaxCeArgs()
    a.dim, a.n, a.vocab, a.scale = 16, 4, vocab, 1.0
    setattr(a, which, 64)
    assert getattr(_lib.lib, name)(C.byref(a), None) != 0  # (in range: an array is NULL)
    assert (b"out of range" in _lib.lib.mono_last_error()) == refused
    assert (getattr(_lib.lib, name + "_workspace")(C.byref(a)) == -1) == refused
    setattr(a, which, None)
    a.grad_query = 64
    assert getattr(_lib.lib, name + "_workspace")(C.byref(a)) >= 0


@pytest.mark.parametrize("leaf", ["rows", "bias"])
def test_the_entry_point_refuses_before_the_forward(leaf):
  rows, bias = torch.zeros(1, 1), torch.zeros(1)
  if leaf == "rows":
    rows.requires_grad_()
  else:
    bias.requires_grad_()
  with pytest.raises(ValueError, match="too many"):
    loss_ops.softmax_cross_entropy(torch.zeros(2, 1), rows.expand(MOST, 1), torch.zeros(2, dtype=torch.int64),
                                   bias.expand(MOST))


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_most_queries(dtype):
  """2^26 - 1 of them, every loss and every query's gradient against 64 bits. Magnitudes S of the logits are below
  20, so a weight is off by e = 2^-23 (5 S + 6 (S + 2) + 15) = 3e-5 of itself."""
  n, gen = 2 ** 26 - 1, torch.Generator(device="cuda").manual_seed(0)
  q = torch.randn(n, 1, generator=gen, device="cuda").to(dtype).requires_grad_()
  w = torch.tensor([[1.0], [-2.0], [0.5]], device="cuda", dtype=dtype)
  labels = torch.randint(0, 3, (n,), generator=gen, device="cuda")
  loss = loss_ops.softmax_cross_entropy(q, w, labels)
  grad, = torch.autograd.grad(loss, q, torch.ones_like(loss))
  half, e = (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24), 3e-5
  for at in range(0, n, 2 ** 23):
    part = slice(at, min(n, at + 2 ** 23))
    x = q.detach()[part].double() @ w.double().t()
    assert x.abs().max() < 20
    d = torch.softmax(x, 1)
    want = torch.logsumexp(x, 1) - x.gather(1, labels[part, None])[:, 0]
    assert ((loss.detach()[part].double() - want).abs() <= e + 8 * 2.0 ** -24 * want).all()
    d.scatter_add_(1, labels[part, None], torch.full_like(x[:, :1], -1.0))
    want = d @ w.double()
    off = (half + e) * (d.abs() @ w.double().abs())
    assert ((grad[part].double() - want).abs() <= off + half * (want.abs() + off)).all()
