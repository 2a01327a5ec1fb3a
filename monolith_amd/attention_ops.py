"""Attention over ragged embedding rows: what a sequential recommender does between the first N
embeddings of a behaviour slot and its dense layers. It stands beside the pooling ops of
distribution_ops.py (a query-weighted mean in place of reduce_sum / reduce_mean) and has no
counterpart in the reference's op set.

Rows are float32 or bfloat16 tensors [n, heads, dim] with dim <= 128 (a 2-D [n, dim] tensor is one
head); the sequences of a batch lie one behind the other and are given by int64 splits
[batch + 1] on the same device, as in embedding_combiners.Ragged: non-decreasing, inside [0, n].
Rows in front of the first split and behind the last (the padding of a fixed-size buffer) belong to
no sequence: their outputs and gradients are zero. Splits that break this give wrong values, never
an access outside the tensors. Softmax statistics and sums are held in 32 bits; results have the
rows' type and are the same bit for bit from call to call. Weights of bfloat16 rows are rounded to
bfloat16 for the product with the values, as are the gradient's for its products. Elements that a query
sees have to be finite (float32 rows are multiplied as three bfloat16 numbers each; an infinite element
gives NaN). The log-sum that the gradient reads is a 32-bit number: its weights are off by
2^-23 |scale * query . key| of themselves, and where that product passes 2^31 the softmax itself gives
NaN. Nothing synchronises the host, and scratch memory comes from torch's allocator, so every op can be
captured into a HIP graph. There is no forward-mode derivative: a tangent (torch.autograd.forward_ad) is
refused."""
import math
from typing import Optional

import torch

from monolith_amd import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}  # MONO_ROW_*
MAX_DIM = 128


def _heads(x: torch.Tensor, name: str, who: str) -> torch.Tensor:
  """[n, heads, dim] with the last dimension contiguous."""
  if not isinstance(x, torch.Tensor) or x.dim() not in (2, 3):
    raise ValueError("%s: %s must be a [n, heads, dim] or [n, dim] tensor" % (who, name))
  if x.dim() == 2:
    x = x.unsqueeze(1)
  return x if x.stride(2) == 1 else x.contiguous()


def _query(query, who):
  q = _heads(query, "query", who)
  if q.dtype not in _DTYPES:
    raise ValueError("%s: rows must be float32 or bfloat16, got %s" % (who, q.dtype))
  if not 1 <= q.shape[2] <= MAX_DIM:
    raise ValueError("%s: dim must be in [1, %d], got %d" % (who, MAX_DIM, q.shape[2]))
  if q.shape[1] < 1:
    raise ValueError("%s: query has no heads" % who)
  return q


def _keys(q, key, value, who, name=""):
  k = _heads(key, name + "key", who)
  v = k if value is None else _heads(value, name + "value", who)
  dtype, device = q.dtype, q.device
  for x in (k,) if v is k else (k, v):
    if x.dtype != dtype or x.device != device:
      raise ValueError("%s: %s is %s on %s, query is %s on %s" % (
          who, name + ("key" if x is k else "value"), x.dtype, x.device, dtype, device))
  shape = k.shape
  if v is not k and v.shape != shape:
    raise ValueError("%s: %svalue %s is not shaped like %skey %s" % (who, name, tuple(v.shape), name,
                                                                   tuple(shape)))
  if shape[2] != q.shape[2]:
    raise ValueError("%s: %skey has dim %d, query %d" % (who, name, shape[2], q.shape[2]))
  if shape[1] < 1 or q.shape[1] % shape[1]:
    raise ValueError("%s: %d query heads are no multiple of %d key heads" % (who, q.shape[1], shape[1]))
  return k, v


def _splits(x, n_batch, device, name: str, who: str) -> torch.Tensor:
  if not isinstance(x, torch.Tensor) or x.dim() != 1 or x.numel() < 1 or \
      x.dtype not in (torch.int64, torch.int32):
    raise ValueError("%s: %s must be an int64 vector [batch + 1]" % (who, name))
  if x.device != device:
    raise ValueError("%s: %s is on %s, query on %s" % (who, name, x.device, device))
  if n_batch is not None and x.numel() != n_batch + 1:
    raise ValueError("%s: %s has %d entries for a batch of %d" % (who, name, x.numel(), n_batch))
  return x if x.dtype == torch.int64 and x.is_contiguous() else x.to(torch.int64).contiguous()


def _mask(x, n, device, name: str, who: str) -> Optional[torch.Tensor]:
  if x is None:
    return None
  if x.dtype != torch.bool or x.dim() != 1 or x.numel() != n or x.device != device:
    raise ValueError("%s: %s must be a bool vector of %d entries on %s" % (who, name, n, device))
  return x.contiguous()


def _scale(scale, dim, who) -> float:
  if scale is None:
    return 1.0 / math.sqrt(dim)
  scale = float(scale)
  if not 1e-20 <= scale <= 1e20:
    raise ValueError("%s: scale must be in [1e-20, 1e20], got %r" % (who, scale))
  return scale


def _on_gpu(x: torch.Tensor, who: str):
  if not x.is_cuda:
    raise _lib.MonolithHipError("%s: tensors must live on the GPU (no CPU fallback)" % who)


_NO_ROWS = (0, 0, 0)


def _rows(x: Optional[torch.Tensor]):
  return _NO_ROWS if x is None else (x.data_ptr(), x.stride(0), x.stride(1))


def _ptr(x: Optional[torch.Tensor]) -> int:
  return 0 if x is None else x.data_ptr()


def _fields(q, k, v, key_splits, query_splits, key_mask, causal, scale, out, rest, lse, kv_heads=None,
            prefix=(0, _NO_ROWS, _NO_ROWS, 0), backward=(0, _NO_ROWS, 0, 0, 0)):
  """The fields of mono_attention_args up to the workspace."""
  nq, heads, dim = q.shape
  splits = key_splits if key_splits is not None else query_splits
  key = _rows(k)
  shared, grad_out, dq, dk, dv = backward
  n_prefix, prefix_key, prefix_value, prefix_mask = prefix
  return (_DTYPES[q.dtype], heads, k.shape[1] if kv_heads is None else kv_heads, dim, causal, shared,
          nq if splits is None else splits.numel() - 1, nq, 0 if k is None else k.shape[0],
          *_rows(q), *key, *(key if v is k else _rows(v)),
          _ptr(query_splits), _ptr(key_splits), _ptr(key_mask), scale,
          n_prefix, *prefix_key, *prefix_value, prefix_mask, out.data_ptr(), _ptr(rest), _ptr(lse),
          *grad_out, dq, dk, dv)


def _forward(q, k, v, key_splits, query_splits, key_mask, causal, scale, for_backward):
  device = q.device
  out = torch.empty(q.shape, dtype=q.dtype, device=device)
  lse = rest = None
  if for_backward:
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=device)
    if q.dtype == torch.bfloat16:
      rest = torch.empty_like(out)
  _lib.launch("mono_ragged_attention", _lib.pack_attention,
              _fields(q, k, v, key_splits, query_splits, key_mask, causal, scale, out, rest, lse), device)
  return out, lse, rest


class _RaggedAttention(torch.autograd.Function):

  @staticmethod
  def forward(ctx, query, key, value, key_splits, query_splits, key_mask, causal, scale):
    v = key if value is None else value
    out, lse, rest = _forward(query, key, v, key_splits, query_splits, key_mask, causal, scale, True)
    ctx.save_for_backward(query, key, value, key_splits, query_splits, key_mask, out, lse, rest)
    ctx.causal, ctx.scale = causal, scale
    return out

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, grad):
    query, key, value, key_splits, query_splits, key_mask, out, lse, rest = ctx.saved_tensors
    shared = value is None
    _lib.no_tangents("the gradient of ragged_attention", grad)
    grad = grad if grad.stride(2) == 1 and grad.dtype == query.dtype else \
        grad.to(query.dtype).contiguous()
    dq = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    dk = dv = None
    if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
      dk = torch.empty(key.shape, dtype=key.dtype, device=key.device)
      if not shared:
        dv = torch.empty(value.shape, dtype=value.dtype, device=value.device)
    _lib.launch("mono_ragged_attention_gradient", _lib.pack_attention,
                _fields(query, key, key if shared else value, key_splits, query_splits, key_mask,
                        ctx.causal, ctx.scale, out, rest, lse,
                        backward=(shared, _rows(grad), dq.data_ptr(), _ptr(dk), _ptr(dv))),
                query.device)
    return dq, dk, dv, None, None, None, None, None


def ragged_attention(query: torch.Tensor, key: torch.Tensor, value: Optional[torch.Tensor],
                     key_splits: torch.Tensor, query_splits: Optional[torch.Tensor] = None,
                     key_mask: Optional[torch.Tensor] = None, causal: bool = False,
                     scale: Optional[float] = None) -> torch.Tensor:
  """out[i, h] = sum_j p_j value[j, h'] with p the softmax over the allowed keys j of i's sequence of
  scale * query[i, h] . key[j, h'], h' = h // (heads // kv_heads). Differentiable in query, key and
  value; the backward recomputes p from one stored number per (query, head).

  query [n_query, heads, dim]; key, value [n_key, kv_heads, dim], value=None: the keys are the values
  too (pooling), and their gradient is the sum of both. key_splits [batch + 1]; query_splits
  [batch + 1], or None: query i belongs to sequence i. key_mask: bool [n_key], False = nobody sees
  this key, whatever its rows hold (an id the table does not have). causal: a sequence's last query
  stands at its last key and sees no key behind its own. scale: 1 / sqrt(dim) by default. A query
  without any allowed key gets zeros and passes no gradient on."""
  who = "ragged_attention"
  q = _query(query, who)
  k, v = _keys(q, key, value, who)
  if key_splits is None:
    raise ValueError("%s: key_splits is missing" % who)
  n_batch = q.shape[0] if query_splits is None else None
  ks = _splits(key_splits, n_batch, q.device, "key_splits", who)
  qs = None if query_splits is None else _splits(query_splits, ks.numel() - 1, q.device,
                                                 "query_splits", who)
  mask = _mask(key_mask, k.shape[0], q.device, "key_mask", who)
  scale = _scale(scale, q.shape[2], who)
  _lib.no_tangents(who, q, k, v)
  _on_gpu(q, who)
  if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
    out = _RaggedAttention.apply(q, k, None if value is None else v, ks, qs, mask, bool(causal),
                                 scale)
  else:
    out = _forward(q, k, v, ks, qs, mask, bool(causal), scale, False)[0]
  return out.view(query.shape) if query.dim() == 2 else out


def shared_prefix_attention(query: torch.Tensor, prefix_key: torch.Tensor,
                            prefix_value: Optional[torch.Tensor],
                            key: Optional[torch.Tensor] = None,
                            value: Optional[torch.Tensor] = None,
                            key_splits: Optional[torch.Tensor] = None,
                            query_splits: Optional[torch.Tensor] = None,
                            prefix_mask: Optional[torch.Tensor] = None,
                            key_mask: Optional[torch.Tensor] = None, causal: bool = False,
                            scale: Optional[float] = None) -> torch.Tensor:
  """Serving: many candidates scored against one user's history. Every query attends to the prefix
  rows, which lie in memory once for the whole batch and are read once for all of it, and to the
  keys of its own sequence, in one softmax. Forward only.

  prefix_key, prefix_value [n_prefix, kv_heads, dim]; the other arguments as in ragged_attention;
  key=None: no keys of their own (with query_splits, queries outside of them see no prefix either and get
  zeros). causal concerns a sequence's own keys, which stand behind the
  prefix; prefix_mask: bool [n_prefix]. value=None / prefix_value=None: the keys are the values."""
  who = "shared_prefix_attention"
  q = _query(query, who)
  pk, pv = _keys(q, prefix_key, prefix_value, who, "prefix_")
  k = v = ks = None
  if key is not None:
    k, v = _keys(q, key, value, who)
    if k.shape[1] != pk.shape[1]:
      raise ValueError("%s: key has %d heads, prefix_key %d" % (who, k.shape[1], pk.shape[1]))
    if key_splits is None:
      raise ValueError("%s: key_splits is missing" % who)
    ks = _splits(key_splits, q.shape[0] if query_splits is None else None, q.device, "key_splits", who)
  elif value is not None or key_splits is not None or key_mask is not None:
    raise ValueError("%s: value, key_splits and key_mask need a key" % who)
  qs = None if query_splits is None else _splits(
      query_splits, None if ks is None else ks.numel() - 1, q.device, "query_splits", who)
  if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, pk, pv, k, v)):
    raise ValueError("%s has no gradient: detach the tensors or use ragged_attention" % who)
  _lib.no_tangents(who, q, pk, pv, k, v)
  scale = _scale(scale, q.shape[2], who)
  mask = None if k is None else _mask(key_mask, k.shape[0], q.device, "key_mask", who)
  pmask = _mask(prefix_mask, pk.shape[0], q.device, "prefix_mask", who)
  _on_gpu(q, who)
  out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
  _lib.launch("mono_shared_prefix_attention", _lib.pack_attention,
              _fields(q, k, v, ks, qs, mask, bool(causal), scale, out, None, None, kv_heads=pk.shape[1],
                      prefix=(pk.shape[0], _rows(pk), _rows(pv), _ptr(pmask))), q.device)
  return out.view(query.shape) if query.dim() == 2 else out
