"""Softmax cross entropy against embedding rows: the loss of a retrieval or next-item model whose
output layer is a hash table. The candidates are rows that HashTable.lookup returned, the gradient
of the rows goes to HashTable.apply_gradients, and the bias takes the correction for how often a
candidate is drawn (what a table under entry.BatchSoftmaxOptimizer estimates). No counterpart in
the reference's op set.

The logits [n, vocab] never exist in memory. Sums and statistics are held in 32 bits; in the gradient of bfloat16 rows
the probabilities, the label's p - 1 in the rows' gradient among them, are rounded to bfloat16 for the products. Rows
are to be finite. The log-sum that the gradient reads is a 32-bit number: its probabilities are off by 2^-23 |logit| of
themselves, and where logits pass 2^31 the loss is NaN. Results are the same bit for bit from call to call. Nothing synchronises the host and scratch memory comes from
torch's allocator, so loss and gradient can be captured into a HIP graph. There is no forward-mode
derivative: a tangent (torch.autograd.forward_ad) is refused."""
from typing import Optional

import torch

from monolith_amd import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}  # MONO_ROW_*
MAX_DIM = 256


def _fields(query, rows, labels, bias, scale, loss, lse, grad_loss=0, dq=0, dw=0, db=0):
  """The fields of mono_softmax_ce_args up to the workspace."""
  return (_DTYPES[query.dtype], query.shape[1], query.shape[0], rows.shape[0],
          query.data_ptr(), query.stride(0), rows.data_ptr(), rows.stride(0),
          labels.data_ptr(), 0 if bias is None else bias.data_ptr(), scale, loss, lse.data_ptr(),
          grad_loss, dq, dw, db)


def _forward(query, rows, labels, bias, scale):
  loss = torch.empty(query.shape[0], dtype=torch.float32, device=query.device)
  lse = torch.empty(2 * query.shape[0], dtype=torch.float32, device=query.device)  # log-sums, 1 - p of the labels
  _lib.launch("mono_softmax_cross_entropy", _lib.pack_softmax_ce,
              _fields(query, rows, labels, bias, scale, loss.data_ptr(), lse), query.device)
  return loss, lse


class _SoftmaxCrossEntropy(torch.autograd.Function):

  @staticmethod
  def forward(ctx, query, rows, labels, bias, scale):
    loss, lse = _forward(query, rows, labels, bias, scale)
    ctx.save_for_backward(query, rows, labels, bias, lse)
    ctx.scale = scale
    return loss

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, grad):
    query, rows, labels, bias, lse = ctx.saved_tensors
    _lib.no_tangents("the gradient of softmax_cross_entropy", grad)
    if grad.dtype != torch.float32 or not grad.is_contiguous():
      grad = grad.to(torch.float32).contiguous()
    dq = dw = db = None
    ptrs = [0, 0, 0]
    if ctx.needs_input_grad[0]:
      dq = torch.empty(query.shape, dtype=query.dtype, device=query.device)
      ptrs[0] = dq.data_ptr()
    if ctx.needs_input_grad[1]:
      dw = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
      ptrs[1] = dw.data_ptr()
    if bias is not None and ctx.needs_input_grad[3]:
      db = torch.empty_like(bias)
      ptrs[2] = db.data_ptr()
    _lib.launch("mono_softmax_cross_entropy_gradient", _lib.pack_softmax_ce,
                _fields(query, rows, labels, bias, ctx.scale, 0, lse, grad.data_ptr(), *ptrs),
                query.device)
    return dq, dw, None, db, None


def softmax_cross_entropy(query: torch.Tensor, rows: torch.Tensor, labels: torch.Tensor,
                          bias: Optional[torch.Tensor] = None, scale: float = 1.0) -> torch.Tensor:
  """loss[i] = log sum_v exp(l[i, v]) - l[i, labels[i]], l = scale * query rows^T + bias; float32 [n],
  not reduced. Differentiable in query, rows and bias.

  query [n, dim], rows [vocab, dim]: float32 or bfloat16, dim <= 256; labels int64 [n]: a label of -1
  marks a query without one (loss 0, no gradient), any other label outside [0, vocab) gives a loss of
  NaN and no gradient. bias: float32 [vocab]; -inf takes a candidate out, whatever its row holds, and
  a query whose own label is taken out has a loss of +inf and no gradient; a finite bias below -1e7
  counts as -1e7 beside the other candidates. scale: 1 / temperature."""
  who = "softmax_cross_entropy"
  for name, x in (("query", query), ("rows", rows)):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
      raise ValueError("%s: %s must be a matrix" % (who, name))
  if query.dtype not in _DTYPES:
    raise ValueError("%s: rows must be float32 or bfloat16, got %s" % (who, query.dtype))
  if rows.dtype != query.dtype or rows.device != query.device:
    raise ValueError("%s: rows are %s on %s, query is %s on %s" % (who, rows.dtype, rows.device,
                                                                   query.dtype, query.device))
  if rows.shape[1] != query.shape[1] or not 1 <= query.shape[1] <= MAX_DIM:
    raise ValueError("%s: dim must be the same and in [1, %d], got query %s, rows %s" % (
        who, MAX_DIM, tuple(query.shape), tuple(rows.shape)))
  if rows.shape[0] < 1:
    raise ValueError("%s: there are no rows" % who)
  if query.shape[0] >= 2 ** 26:
    raise ValueError("%s: %d queries are too many for one call" % (who, query.shape[0]))
  if not isinstance(labels, torch.Tensor) or labels.dtype != torch.int64 or \
      labels.shape != query.shape[:1] or labels.device != query.device:
    raise ValueError("%s: labels must be an int64 vector [%d] on %s" % (who, query.shape[0],
                                                                       query.device))
  if bias is not None and (bias.dtype != torch.float32 or bias.shape != rows.shape[:1] or
                           bias.device != query.device):
    raise ValueError("%s: bias must be a float32 vector [%d] on %s" % (who, rows.shape[0],
                                                                      query.device))
  if rows.shape[0] >= 2 ** 31 - 2 ** 27 and (rows.requires_grad or (bias is not None and bias.requires_grad)):
    raise ValueError("%s: %d rows are too many for their gradient" % (who, rows.shape[0]))
  scale = float(scale)
  if not 1e-20 <= scale <= 1e20:
    raise ValueError("%s: scale must be in [1e-20, 1e20], got %r" % (who, scale))
  _lib.no_tangents(who, query, rows, bias)
  if not query.is_cuda:
    raise _lib.MonolithHipError("%s: tensors must live on the GPU (no CPU fallback)" % who)
  query = query if query.stride(1) == 1 else query.contiguous()
  rows = rows if rows.stride(1) == 1 else rows.contiguous()
  labels = labels.contiguous()
  bias = None if bias is None else bias.contiguous()
  if torch.is_grad_enabled() and (query.requires_grad or rows.requires_grad or
                                  (bias is not None and bias.requires_grad)):
    return _SoftmaxCrossEntropy.apply(query, rows, labels, bias, scale)
  return _forward(query, rows, labels, bias, scale)[0]
