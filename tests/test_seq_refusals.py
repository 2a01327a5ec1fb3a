"""CPU: what the sequence and loss operators refuse, at the Python entry points and at the C ABI, before
anything is launched; and the restated gradients (tests/seq_ref.py) against differences."""
import ctypes as C

import numpy as np
import pytest
import torch

from monolith_amd import _lib, attention_ops, loss_ops
from tests import seq_ref


def _att(**kw):
  a = dict(query=torch.zeros(6, 4, 16), key=torch.zeros(9, 2, 16), value=torch.zeros(9, 2, 16),
           key_splits=torch.tensor([0, 4, 9]), query_splits=torch.tensor([0, 2, 6]))
  a.update(kw)
  return attention_ops.ragged_attention(**a)


BAD_ATTENTION = [
    dict(query=torch.zeros(6)), dict(query=torch.zeros(6, 4, 16, 1)), dict(query=None),
    dict(query=torch.zeros(6, 4, 16, dtype=torch.float16)),
    dict(query=torch.zeros(6, 4, 16, dtype=torch.float64)),
    dict(query=torch.zeros(6, 4, 129), key=torch.zeros(9, 2, 129), value=None),
    dict(query=torch.zeros(6, 4, 0), key=torch.zeros(9, 2, 0), value=None),
    dict(query=torch.zeros(6, 0, 16)), dict(query=torch.zeros(6, 3, 16)),
    dict(key=torch.zeros(9, 0, 16), value=None), dict(key=torch.zeros(9, 2, 8), value=None),
    dict(key=torch.zeros(9, 2, 16, dtype=torch.bfloat16)), dict(value=torch.zeros(9, 1, 16)),
    dict(value=torch.zeros(8, 2, 16)), dict(value=torch.zeros(9, 2, 16, dtype=torch.bfloat16)),
    dict(key_splits=None), dict(key_splits=[0, 4, 9]), dict(key_splits=torch.tensor([0.0, 4.0, 9.0])),
    dict(key_splits=torch.zeros(0, dtype=torch.int64)), dict(key_splits=torch.zeros(3, 1, dtype=torch.int64)),
    dict(query_splits=torch.tensor([0, 6])), dict(query_splits=None),
    dict(key_mask=torch.ones(8, dtype=torch.bool)), dict(key_mask=torch.ones(9)),
    dict(key_mask=torch.ones(9, 1, dtype=torch.bool)),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-21),
]


@pytest.mark.parametrize("i", range(len(BAD_ATTENTION)))
def test_ragged_attention_refuses(i):
  with pytest.raises(ValueError):
    _att(**BAD_ATTENTION[i])


def _pre(**kw):
  a = dict(query=torch.zeros(6, 4, 16), prefix_key=torch.zeros(5, 2, 16), prefix_value=torch.zeros(5, 2, 16),
           key=torch.zeros(9, 2, 16), value=torch.zeros(9, 2, 16), key_splits=torch.tensor([0, 4, 9]),
           query_splits=torch.tensor([0, 2, 6]))
  a.update(kw)
  return attention_ops.shared_prefix_attention(**a)


BAD_PREFIX = [
    dict(prefix_key=None), dict(prefix_key=torch.zeros(5, 3, 16)), dict(prefix_value=torch.zeros(4, 2, 16)),
    dict(prefix_key=torch.zeros(5, 1, 16), prefix_value=None), dict(key_splits=None),
    dict(key=None), dict(key=None, value=None), dict(prefix_mask=torch.ones(4, dtype=torch.bool)),
    dict(query=torch.zeros(6, 4, 16, requires_grad=True)),
    dict(prefix_key=torch.zeros(5, 2, 16, requires_grad=True)), dict(query_splits=torch.tensor([0, 6])),
    dict(query_splits=None),
]


@pytest.mark.parametrize("i", range(len(BAD_PREFIX)))
def test_shared_prefix_attention_refuses(i):
  with pytest.raises(ValueError):
    _pre(**BAD_PREFIX[i])


def _ce(**kw):
  a = dict(query=torch.zeros(6, 16), rows=torch.zeros(9, 16), labels=torch.zeros(6, dtype=torch.int64),
           bias=torch.zeros(9))
  a.update(kw)
  return loss_ops.softmax_cross_entropy(**a)


BAD_CE = [
    dict(query=None), dict(query=torch.zeros(6, 1, 16)), dict(rows=torch.zeros(9)),
    dict(query=torch.zeros(6, 16, dtype=torch.float16), rows=torch.zeros(9, 16, dtype=torch.float16)),
    dict(rows=torch.zeros(9, 16, dtype=torch.bfloat16)), dict(rows=torch.zeros(9, 15)),
    dict(query=torch.zeros(6, 257), rows=torch.zeros(9, 257)), dict(query=torch.zeros(6, 0), rows=torch.zeros(9, 0)),
    dict(rows=torch.zeros(0, 16), bias=None), dict(labels=torch.zeros(5, dtype=torch.int64)),
    dict(labels=torch.zeros(6, dtype=torch.int32)), dict(labels=torch.zeros(6, 1, dtype=torch.int64)),
    dict(labels=[0] * 6), dict(bias=torch.zeros(8)), dict(bias=torch.zeros(9, dtype=torch.float64)),
    dict(scale=0.0), dict(scale=-2.0), dict(scale=float("inf")), dict(scale=float("nan")),
]


@pytest.mark.parametrize("i", range(len(BAD_CE)))
def test_softmax_cross_entropy_refuses(i):
  with pytest.raises(ValueError):
    _ce(**BAD_CE[i])


def test_cpu_tensors_are_refused():
  for call in (_att, _pre, _ce):
    with pytest.raises(_lib.MonolithHipError, match="no CPU fallback"):
      call()


def _c_attention(**kw):
  a = _lib.AttentionArgs()
  a.heads = a.kv_heads = 1
  a.dim, a.batch, a.n_query, a.n_key, a.scale = 16, 2, 2, 5, 1.0
  a.key_splits = 64  # (never read: every call below is refused first)
  for n, v in kw.items():
    setattr(a, n, v)
  return a


BAD_C = [dict(dtype=2), dict(dtype=-1), dict(dim=0), dict(dim=129), dict(heads=0), dict(kv_heads=0),
         dict(heads=3, kv_heads=2), dict(batch=-1), dict(n_query=-1), dict(n_key=-1), dict(n_prefix=-1),
         dict(n_query=3), dict(n_query=2 ** 31, query_splits=64), dict(n_key=2 ** 31), dict(scale=0.0),
         dict(scale=float("nan")), dict(scale=-1.0), dict(scale=float("inf")), dict(workspace=8)]


@pytest.mark.parametrize("i", range(len(BAD_C)))
def test_c_attention_refuses(i):
  a = _c_attention(**BAD_C[i])
  for name in ("mono_ragged_attention", "mono_ragged_attention_gradient", "mono_shared_prefix_attention"):
    assert getattr(_lib.lib, name)(C.byref(a), None) != 0
    assert name.encode() in _lib.lib.mono_last_error()
    assert getattr(_lib.lib, name + "_workspace")(C.byref(a)) == -1


def test_c_small_workspaces_and_missing_pointers_are_refused():
  long = _c_attention(batch=1, n_query=1, n_key=100000)
  assert _lib.lib.mono_ragged_attention_workspace(C.byref(long)) > 0
  assert _lib.lib.mono_ragged_attention_gradient(C.byref(long), None) != 0
  assert b"too small" in _lib.lib.mono_last_error()
  for name in ("mono_ragged_attention", "mono_ragged_attention_gradient"):
    assert getattr(_lib.lib, name)(None, None) != 0
    a = _c_attention(key_splits=None)
    assert getattr(_lib.lib, name)(C.byref(a), None) != 0
    assert b"key_splits" in _lib.lib.mono_last_error()
  for name in ("mono_ragged_attention", "mono_ragged_attention_gradient", "mono_shared_prefix_attention"):
    a = _c_attention(workspace=64, workspace_bytes=2 ** 30)
    assert getattr(_lib.lib, name)(C.byref(a), None) != 0
    assert b"NULL" in _lib.lib.mono_last_error()
  pre = _c_attention(n_prefix=100000)
  pre.query.ptr = pre.out = pre.key.ptr = pre.value.ptr = pre.prefix_key.ptr = pre.prefix_value.ptr = 64
  long.query.ptr = long.out = long.key.ptr = long.value.ptr = 64
  assert _lib.lib.mono_ragged_attention(C.byref(long), None) != 0
  assert b"too small" in _lib.lib.mono_last_error()
  assert _lib.lib.mono_shared_prefix_attention(C.byref(pre), None) != 0
  assert b"too small" in _lib.lib.mono_last_error()


def test_c_cross_entropy_refuses():
  for kw in (dict(dtype=2), dict(dim=0), dict(dim=257), dict(n=-1), dict(vocab=0), dict(vocab=2 ** 31),
             dict(n=2 ** 26), dict(scale=0.0), dict(scale=1e30), dict(workspace=4)):
    a = _lib.SoftmaxCeArgs()
    a.dim, a.n, a.vocab, a.scale = 16, 4, 100, 1.0
    for n, v in kw.items():
      setattr(a, n, v)
    for name in ("mono_softmax_cross_entropy", "mono_softmax_cross_entropy_gradient"):
      assert getattr(_lib.lib, name)(C.byref(a), None) != 0
      assert getattr(_lib.lib, name + "_workspace")(C.byref(a)) == -1
  a = _lib.SoftmaxCeArgs()
  a.dim, a.n, a.vocab, a.scale = 16, 40, 100000, 1.0
  for name in ("mono_softmax_cross_entropy", "mono_softmax_cross_entropy_gradient"):
    assert getattr(_lib.lib, name)(C.byref(a), None) != 0
    assert b"NULL" in _lib.lib.mono_last_error()
  a.query = a.rows = a.labels = a.loss = a.lse = 64
  assert _lib.lib.mono_softmax_cross_entropy(C.byref(a), None) != 0
  assert b"too small" in _lib.lib.mono_last_error()


def test_packed_arguments_are_the_structures():
  """The packed form that the operators pass is the ctypes.Structure's image, field by field."""
  def image(cls, pack):
    names, kinds = [], []
    for n, t in cls._fields_:
      for m, u in (t._fields_ if issubclass(t, C.Structure) else [(None, t)]):
        names.append((n, m))
        kinds.append(u)
    values = [(0.5 * i if u is C.c_float else i + 1) for i, u in enumerate(kinds)]
    a = cls()
    for (n, m), v in zip(names, values):
      setattr(getattr(a, n) if m else a, m or n, v)
    assert bytes(a) == pack(*values)
  image(_lib.AttentionArgs, _lib.pack_attention)
  image(_lib.SoftmaxCeArgs, _lib.pack_softmax_ce)


def test_structures_have_the_header_s_size():
  assert C.sizeof(_lib.AttentionArgs) == 304 and C.sizeof(_lib.SoftmaxCeArgs) == 144


def test_restated_gradients_against_differences():
  """In 64 bits, h = 1e-5: the cubic term is 1e-10 of a derivative of order 1, the rounding 1e-16 / h."""
  rng = np.random.default_rng(0)
  q, k, v = (rng.standard_normal(s) for s in ((9, 4, 6), (11, 2, 6), (11, 2, 6)))
  g = rng.standard_normal(q.shape)
  segs = seq_ref.segments(np.array([0, 4, 4, 9]), np.array([0, 5, 6, 11]))
  keep = seq_ref.keep_rule(segs, rng.random(11) > 0.2, True)
  ref = lambda x, gg=None: seq_ref.attention(*x, segs, keep, 0.4, "fp32", gg)
  grads = ref([q, k, v], g)
  for i, name in enumerate(("dq", "dk", "dv")):
    u = rng.standard_normal([q, k, v][i].shape)
    x, y = [q, k, v], [q, k, v]
    x[i], y[i] = x[i] + 1e-5 * u, y[i] - 1e-5 * u
    diff = ((ref(x)["out"][0] - ref(y)["out"][0]) * g).sum() / 2e-5
    assert abs(diff - (grads[name][0] * u).sum()) < 1e-7
  q, w, b, g = rng.standard_normal((7, 5)), rng.standard_normal((9, 5)), rng.standard_normal(9), rng.standard_normal(7)
  b[2] = -np.inf
  lab = np.array([0, 3, -1, 8, 8, 1, 4])
  ce = lambda x, gg=None: seq_ref.cross_entropy(x[0], x[1], lab, x[2], 0.7, "fp32", gg)
  grads = ce([q, w, b], g)
  for i, name in enumerate(("dq", "dw", "db")):
    u = rng.standard_normal([q, w, b][i].shape)
    x, y = [q, w, b], [q, w, b]
    x[i], y[i] = x[i] + 1e-5 * u, y[i] - 1e-5 * u
    diff = ((ce(x)["loss"][0] - ce(y)["loss"][0]) * g).sum() / 2e-5
    assert abs(diff - (grads[name][0] * u).sum()) < 1e-7
