"""GPU: the sequence and loss operators at the ends of their range: rows more than 2^31 elements apart, long causal
gradients of wide rows, splits that break their rule."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import seq_ref
from tests.test_attention_gpu import TYPES, dev, on, rows, run_both, splits

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [96, 128])
def test_long_causal_gradients_of_wide_rows(dtype, D):
  rng = np.random.default_rng(D)
  run_both(rng, dtype, 2, 1, D, [1300, 3, 0, 140], [1300, 3, 0, 140], causal=True, mask=0.1)
  run_both(rng, dtype, 2, 2, D, [700], [900], causal=True)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_rows_beyond_two_to_the_31_elements(dtype):
  """300 rows 7 * 2^20 elements apart, the last at more than 2^31: the same results as the rows side by side."""
  from monolith_amd import attention_ops, loss_ops
  rng = np.random.default_rng(1)
  n, step = 300, 7 * 2 ** 20
  room = torch.empty(n * step, dtype=TYPES[dtype], device=dev())
  far = room.as_strided((n, 2, 32), (step, step // 2, 1))
  far.copy_(rows(rng, (n, 2, 32), dtype)[0])
  assert (n - 1) * step > 2 ** 31
  near = far.contiguous()
  s = on(splits([100, 200]))
  labels = on(rng.integers(0, n, n))

  def results(x):
    out = []
    for q, qs in ((x[::150], None), (x, s), (x[::150].repeat(1, 5, 1), None)):
      leaves = [t.detach().requires_grad_() for t in (q, x)]
      got = attention_ops.ragged_attention(*leaves, None, s, qs, causal=True)
      out += [got.detach()] + list(torch.autograd.grad(got, leaves, torch.ones_like(got)))
    out.append(attention_ops.shared_prefix_attention(x, x, None, x, None, s, s))
    leaves = [x[:, 1].detach().requires_grad_(), x[:, 0].detach().requires_grad_()]
    loss = loss_ops.softmax_cross_entropy(*leaves, labels)
    return out + [loss.detach()] + list(torch.autograd.grad(loss.sum(), leaves))

  for a, b in zip(results(far), results(near)):
    assert torch.equal(a, b)


def test_bfloat16_attention_combiner():
  from monolith_amd import embedding_combiners as ec
  rng = np.random.default_rng(2)
  lens = [3, 0, 1, 40, 7]
  s, n, dim, heads = splits(lens), sum(lens), 24, 3
  e, e64 = rows(rng, (n, dim), "bf16")
  q, q64 = rows(rng, (5, dim), "bf16")
  g, g64 = rows(rng, (5, dim), "bf16")
  mask = rng.random(n) > 0.2
  e.requires_grad_()
  q.requires_grad_()
  out = ec.Attention(q, heads, on(mask)).combine(ec.Ragged(torch.arange(n, device=dev()), on(s)), e)
  assert out.dtype == torch.bfloat16
  cut = lambda x: x.reshape(len(x), heads, -1)
  segs = seq_ref.segments(None, s)
  want = seq_ref.attention(cut(q64), cut(e64), cut(e64), segs, seq_ref.keep_rule(segs, mask, False),
                           (dim // heads) ** -0.5, "bf16", cut(g64))
  flat = lambda x: tuple(y.reshape(len(y), -1) for y in x)
  seq_ref.check(out, flat(want["out"]), "out")
  out.backward(g)
  seq_ref.check(q.grad, flat(want["dq"]), "dq")
  seq_ref.check(e.grad, flat(want["dkv"]), "dk")


class Guarded:
  """Tensors of the given shapes, each in the middle of a buffer of a known pattern."""
  PAD = 4096

  def __init__(self):
    self.bufs = []

  def new(self, shape, dtype):
    n = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
    buf = torch.full((n + 2 * self.PAD,), 0x5a, dtype=torch.uint8, device=dev())
    self.bufs.append(buf)
    return buf[self.PAD:self.PAD + n].view(dtype).view(shape)

  def check(self):
    for buf in self.bufs:
      assert (buf[:self.PAD] == 0x5a).all() and (buf[-self.PAD:] == 0x5a).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads,form", [(2, "one"), (10, "one"), (2, "many"), (2, "prefix"), (10, "prefix_one")])
@pytest.mark.parametrize("nk", [90, 5000])
def test_broken_splits_stay_inside(dtype, heads, form, nk):
  """Splits that fall or leave [0, rows] give wrong values, but nothing outside of the results is written: results and
  workspace lie between guards. (Every split is held to [0, rows] where it is read, and a sequence that ends before it
  starts has no rows, so every row and part has its place.)"""
  from monolith_amd import _lib, attention_ops as ao
  rng = np.random.default_rng(nk + heads)
  one = form.endswith("one")
  B, D, prefix = 7, 16, 64 if form.startswith("prefix") else 0
  nq = B if one else 200
  q, _ = rows(rng, (nq, heads, D), dtype)
  k, _ = rows(rng, (nk, 2, D), dtype)
  g, _ = rows(rng, (nq, heads, D), dtype)
  pk, _ = rows(rng, (prefix, 2, D), dtype)
  room = Guarded()

  def call(name, fields):
    fn, size = _lib._seq_fns[name]
    n = size(_lib.pack_attention(*fields, 0, 0))
    assert n >= 0
    ws = room.new((n,), torch.uint8)
    _lib.check(fn(_lib.pack_attention(*fields, ws.data_ptr(), n), C.c_void_p(torch.cuda.current_stream().cuda_stream)))

  for trial in range(6):
    ks = on(rng.integers(-nk, 2 * nk, B + 1) if trial else np.array([nk, 0] * 4))
    qs = None if one else on(rng.integers(-nq, 2 * nq, B + 1))
    out, lse = room.new(q.shape, q.dtype), room.new((nq, heads), torch.float32)
    rest = room.new(q.shape, q.dtype) if dtype == "bf16" and not prefix else None
    if prefix:
      call("mono_shared_prefix_attention",
           ao._fields(q, k, k, ks, qs, None, True, 0.25, out, None, None, kv_heads=2,
                      prefix=(prefix, ao._rows(pk), ao._rows(pk), 0)))
    else:
      call("mono_ragged_attention", ao._fields(q, k, k, ks, qs, None, True, 0.25, out, rest, lse))
      dq, dk = room.new(q.shape, q.dtype), room.new(k.shape, k.dtype)
      call("mono_ragged_attention_gradient",
           ao._fields(q, k, k, ks, qs, None, True, 0.25, out, rest, lse,
                      backward=(True, ao._rows(g), dq.data_ptr(), dk.data_ptr(), 0)))
    torch.cuda.synchronize()
    room.check()


@pytest.mark.parametrize("D", [16, 128])
def test_worst_products_of_fp32_rows(D):
  """x = 1 + 2^-8 + 2^-16 has three bf16 parts of one bit each, and what the six products of x * x leave out is
  2 * 2^-24 of it, in every element the same way: a logit of D of them is 2^-23 too small and rounds at most D + 8
  times on the way to the loss, log(1 + exp(l)) = l for an l of more than 17 below a candidate of zeros."""
  from monolith_amd import loss_ops
  x = 1 + 2.0 ** -8 + 2.0 ** -16
  q = torch.full((40, D), x, device=dev())
  w = torch.zeros(2, D, device=dev())
  w[0] = x
  want = D * x * x * 2  # (scale 2; exp(-32) is under 2^-46)
  loss = loss_ops.softmax_cross_entropy(q, w, torch.ones(40, dtype=torch.int64, device=dev()), scale=2.0).double()
  off = (loss / want - 1).abs().max().item()
  assert off <= 2.0 ** -23 + (D + 8) * seq_ref.U32, off


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("scale", [1e-20, 1e20])
def test_scales_at_their_ends(dtype, scale):
  """Rows that much larger or smaller, so that the logits are ordinary: the bounds do not depend on the scale."""
  from monolith_amd import attention_ops, loss_ops
  rng = np.random.default_rng(3)
  size = scale ** -0.5
  lens = [50, 90]
  s = on(splits(lens))
  segs = seq_ref.segments(splits(lens), splits(lens))
  q, q64 = rows(rng, (140, 2, 16), dtype, size)
  k, k64 = rows(rng, (140, 1, 16), dtype, size)
  v, v64 = rows(rng, (140, 1, 16), dtype)
  g, g64 = rows(rng, (140, 2, 16), dtype)
  leaves = [t.requires_grad_() for t in (q, k, v)]
  out = attention_ops.ragged_attention(*leaves, s, s, scale=scale)
  want = seq_ref.attention(q64, k64, v64, segs, seq_ref.keep_rule(segs, None, False), scale, dtype, g64)
  for got, name in zip([out] + list(torch.autograd.grad(out, leaves, g)), ("out", "dq", "dk", "dv")):
    seq_ref.check(got, want[name], name)
  w, w64 = rows(rng, (300, 16), dtype, size)
  labels, bias = rng.integers(0, 300, 140), rng.standard_normal(300).astype(np.float32)
  b = on(bias).requires_grad_()
  leaves = [q[:, 0].detach().requires_grad_(), w.requires_grad_(), b]
  loss = loss_ops.softmax_cross_entropy(leaves[0], w, on(labels), b, scale)
  gl = rng.standard_normal(140).astype(np.float32)
  want = seq_ref.cross_entropy(q64[:, 0], w64, labels, bias.astype(np.float64), scale, dtype, gl.astype(np.float64))
  for got, name in zip([loss] + list(torch.autograd.grad(loss, leaves, on(gl))), ("loss", "dq", "dw", "db")):
    seq_ref.check(got, want[name], name)
