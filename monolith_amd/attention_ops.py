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
rows' type and are the same bit for bit from call to call. Nothing synchronises the host, and
scratch memory comes from torch's allocator, so every op can be captured into a HIP graph."""
import ctypes as C
import math
from typing import Optional

import torch

from monolith_amd import _lib
from monolith_amd._lib import vp

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}  # MONO_ROW_*
MAX_DIM = 128


def _heads(x: torch.Tensor, name: str, who: str) -> torch.Tensor:
  """[n, heads, dim] with the last dimension contiguous."""
  if not isinstance(x, torch.Tensor) or x.dim() not in (2, 3):
    raise ValueError("%s: %s must be a [n, heads, dim] or [n, dim] tensor" % (who, name))
  if x.dim() == 2:
    x = x.unsqueeze(1)
  return x if x.stride(2) == 1 else x.contiguous()


def _same(x: torch.Tensor, like: torch.Tensor, name: str, who: str):
  if x.device != like.device or x.dtype != like.dtype:
    raise ValueError("%s: %s is %s on %s, query is %s on %s" % (who, name, x.dtype, x.device,
                                                                like.dtype, like.device))


def _splits(x, n_batch, device, name: str, who: str) -> torch.Tensor:
  if not isinstance(x, torch.Tensor) or x.dim() != 1 or x.numel() < 1 or \
      x.dtype not in (torch.int64, torch.int32):
    raise ValueError("%s: %s must be an int64 vector [batch + 1]" % (who, name))
  if x.device != device:
    raise ValueError("%s: %s is on %s, query on %s" % (who, name, x.device, device))
  if n_batch is not None and x.numel() != n_batch + 1:
    raise ValueError("%s: %s has %d entries for a batch of %d" % (who, name, x.numel(), n_batch))
  return x.to(torch.int64).contiguous()


def _mask(x, n, device, name: str, who: str) -> Optional[torch.Tensor]:
  if x is None:
    return None
  if x.dtype != torch.bool or x.dim() != 1 or x.numel() != n or x.device != device:
    raise ValueError("%s: %s must be a bool vector of %d entries on %s" % (who, name, n, device))
  return x.contiguous()


def _scale(scale, dim, who) -> float:
  scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
  if not (math.isfinite(scale) and scale > 0):
    raise ValueError("%s: scale must be a positive finite number, got %r" % (who, scale))
  return scale


def _on_gpu(x: torch.Tensor, who: str):
  if not x.is_cuda:
    raise _lib.MonolithHipError("%s: tensors must live on the GPU (no CPU fallback)" % who)


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
  _same(k, q, name + "key", who)
  v = k if value is None else _heads(value, name + "value", who)
  _same(v, q, name + "value", who)
  if v.shape != k.shape:
    raise ValueError("%s: %svalue %s is not shaped like %skey %s" % (who, name, tuple(v.shape), name,
                                                                   tuple(k.shape)))
  if k.shape[2] != q.shape[2]:
    raise ValueError("%s: %skey has dim %d, query %d" % (who, name, k.shape[2], q.shape[2]))
  if k.shape[1] < 1 or q.shape[1] % k.shape[1]:
    raise ValueError("%s: %d query heads are no multiple of %d key heads" % (who, q.shape[1],
                                                                           k.shape[1]))
  return k, v


def _rows(x: torch.Tensor) -> _lib.Rows:
  return _lib.Rows(x.data_ptr(), x.stride(0), x.stride(1))


def _args(q, k, v, key_splits, query_splits, key_mask, causal, scale) -> _lib.AttentionArgs:
  a = _lib.AttentionArgs()
  a.dtype = _DTYPES[q.dtype]
  a.heads, a.dim = q.shape[1], q.shape[2]
  a.causal, a.scale = int(causal), scale
  a.n_query, a.query = q.shape[0], _rows(q)
  a.kv_heads = k.shape[1]
  if key_splits is not None:
    a.n_key, a.key, a.value = k.shape[0], _rows(k), _rows(v)
    a.key_splits = key_splits.data_ptr()
    a.batch = key_splits.numel() - 1
  else:
    a.batch = q.shape[0]
  if query_splits is not None:
    a.query_splits = query_splits.data_ptr()
    a.batch = query_splits.numel() - 1
  if key_mask is not None:
    a.key_mask = key_mask.data_ptr()
  return a


def _call(fn, workspace, a: _lib.AttentionArgs, device) -> None:
  n = workspace(C.byref(a))
  if n < 0:
    _lib.check(1)
  if n:
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
  _lib.launch(fn, a, device)


def _forward(q, k, v, key_splits, query_splits, key_mask, causal, scale, for_backward):
  out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
  lse = rest = None
  a = _args(q, k, v, key_splits, query_splits, key_mask, causal, scale)
  a.out = out.data_ptr()
  if for_backward:
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    a.lse = lse.data_ptr()
    if q.dtype == torch.bfloat16:
      rest = torch.empty_like(out)
      a.out_rest = rest.data_ptr()
  _call(_lib.lib.mono_ragged_attention, _lib.lib.mono_ragged_attention_workspace, a, q.device)
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
    a = _args(query, key, key if shared else value, key_splits, query_splits, key_mask, ctx.causal,
              ctx.scale)
    grad = grad if grad.stride(2) == 1 and grad.dtype == query.dtype else \
        grad.to(query.dtype).contiguous()
    dq = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    a.kv_shared = int(shared)
    a.out, a.lse, a.grad_out = out.data_ptr(), lse.data_ptr(), _rows(grad)
    a.grad_query = dq.data_ptr()
    if rest is not None:
      a.out_rest = rest.data_ptr()
    dk = dv = None
    keys = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
    if keys:
      dk = torch.empty(key.shape, dtype=key.dtype, device=key.device)
      a.grad_key = dk.data_ptr()
    if keys and not shared:
      dv = torch.empty(value.shape, dtype=value.dtype, device=value.device)
      a.grad_value = dv.data_ptr()
    _call(_lib.lib.mono_ragged_attention_gradient,
          _lib.lib.mono_ragged_attention_gradient_workspace, a, query.device)
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
  _on_gpu(q, who)
  if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
    out = _RaggedAttention.apply(q, k, None if value is None else v, ks, qs, mask, bool(causal),
                                 scale)
  else:
    out = _forward(q, k, v, ks, qs, mask, causal, scale, False)[0]
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
  key=None: no keys of their own. causal concerns a sequence's own keys, which stand behind the
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
  scale = _scale(scale, q.shape[2], who)
  mask = None if k is None else _mask(key_mask, k.shape[0], q.device, "key_mask", who)
  pmask = _mask(prefix_mask, pk.shape[0], q.device, "prefix_mask", who)
  _on_gpu(q, who)
  out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
  a = _args(q, pk if k is None else k, pv if k is None else v, ks, qs, mask, causal, scale)
  a.n_prefix, a.prefix_key, a.prefix_value = pk.shape[0], _rows(pk), _rows(pv)
  if pmask is not None:
    a.prefix_mask = pmask.data_ptr()
  a.out = out.data_ptr()
  _call(_lib.lib.mono_shared_prefix_attention, _lib.lib.mono_shared_prefix_attention_workspace, a,
        q.device)
  return out.view(query.shape) if query.dim() == 2 else out
