"""ctypes loader of libmonolith_hip.so. There is no CPU fallback: a missing or unloadable
library raises, and every non-zero status from the C ABI raises MonolithHipError."""
import ctypes as C
import os
import struct

# torch must load its HIP runtime before libmonolith_hip.so pulls in libamdhip64: with the order
# reversed both end up sharing the system copy and torch then reports "No HIP GPUs are available".
import torch  # noqa: F401  pylint: disable=unused-import
from torch.autograd import forward_ad

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmonolith_hip.so")


class MonolithHipError(RuntimeError):
  """Raised for any non-zero status of the C ABI (the reference raises
  tf.errors.InvalidArgumentError / ResourceExhaustedError from its Status)."""


class SegCfg(C.Structure):  # mono_segment_cfg
  _fields_ = [("dim", C.c_int32), ("opt_kind", C.c_int32), ("init_acc", C.c_float),
              ("weight_decay", C.c_float), ("l1", C.c_float), ("l2", C.c_float),
              ("beta", C.c_float), ("init_kind", C.c_int32), ("init_a", C.c_float),
              ("init_b", C.c_float), ("momentum", C.c_float), ("epsilon", C.c_float),
              ("averaging_ratio", C.c_float), ("learning_rate", C.c_float),
              ("use_nesterov", C.c_int32), ("beta1", C.c_float), ("beta2", C.c_float),
              ("comp_kind", C.c_int32), ("comp_a", C.c_float), ("comp_b", C.c_float),
              ("stochastic_rounding_float16", C.c_int32)]


class TableCfg(C.Structure):  # mono_table_cfg
  _fields_ = [("n_segments", C.c_int32), ("default_expire_days", C.c_int32),
              ("segments", C.POINTER(SegCfg)), ("initial_capacity", C.c_int64),
              ("n_slot_expire", C.c_int32), ("entry_type", C.c_int32),
              ("slot_ids", C.POINTER(C.c_int32)), ("slot_expire_days", C.POINTER(C.c_int32)),
              ("seed", C.c_uint64), ("enable_feature_eviction", C.c_int32),
              ("feature_evict_every_n_hours", C.c_int32)]


class Rows(C.Structure):  # mono_rows
  _fields_ = [("ptr", C.c_void_p), ("row_stride", C.c_int64), ("head_stride", C.c_int64)]


class AttentionArgs(C.Structure):  # mono_attention_args
  _fields_ = [("dtype", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32),
              ("dim", C.c_int32), ("causal", C.c_int32), ("kv_shared", C.c_int32),
              ("batch", C.c_int64), ("n_query", C.c_int64), ("n_key", C.c_int64),
              ("query", Rows), ("key", Rows), ("value", Rows), ("query_splits", C.c_void_p),
              ("key_splits", C.c_void_p), ("key_mask", C.c_void_p), ("scale", C.c_float),
              ("n_prefix", C.c_int64), ("prefix_key", Rows), ("prefix_value", Rows),
              ("prefix_mask", C.c_void_p), ("out", C.c_void_p), ("out_rest", C.c_void_p),
              ("lse", C.c_void_p),
              ("grad_out", Rows), ("grad_query", C.c_void_p), ("grad_key", C.c_void_p),
              ("grad_value", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_int64)]


class SoftmaxCeArgs(C.Structure):  # mono_softmax_ce_args
  _fields_ = [("dtype", C.c_int32), ("dim", C.c_int32), ("n", C.c_int64), ("vocab", C.c_int64),
              ("query", C.c_void_p), ("query_stride", C.c_int64), ("rows", C.c_void_p),
              ("rows_stride", C.c_int64), ("labels", C.c_void_p), ("bias", C.c_void_p),
              ("scale", C.c_float), ("loss", C.c_void_p), ("lse", C.c_void_p),
              ("grad_loss", C.c_void_p), ("grad_query", C.c_void_p), ("grad_rows", C.c_void_p),
              ("grad_bias", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_int64)]


_SEQ = ("mono_ragged_attention", "mono_ragged_attention_gradient", "mono_shared_prefix_attention",
        "mono_softmax_cross_entropy", "mono_softmax_cross_entropy_gradient")


def _load():
  if not os.path.exists(LIB_PATH):
    raise ImportError(
        "monolith_amd: %s is missing. Build it with `python -c 'import __graft_entry__ as g; "
        "g.build()'` or `make -C monolith_amd/csrc`; there is no CPU fallback." % LIB_PATH)
  lib = C.CDLL(LIB_PATH)
  lib.mono_last_error.restype = C.c_char_p
  lib.mono_fused_reorder_last_plan.restype = C.c_int64
  for name in _SEQ:
    getattr(lib, name + "_workspace").restype = C.c_int64
  return lib


lib = _load()
_seq_fns = {n: (getattr(lib, n), getattr(lib, n + "_workspace")) for n in _SEQ}


def check(rc):
  if rc != 0:
    raise MonolithHipError((lib.mono_last_error() or b"unknown error").decode())


def vp(x):
  """torch tensor / int / None -> c_void_p."""
  if x is None:
    return C.c_void_p(0)
  if isinstance(x, int):
    return C.c_void_p(x)
  return C.c_void_p(x.data_ptr())


def stream_ptr(device=None):
  import torch
  return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


# The argument structures of the sequence operators, packed in one call: filling a ctypes.Structure field
# by field costs more host time than the launch itself.
pack_attention = struct.Struct("@6i3q" + 3 * "P2q" + "3Pfq" + 2 * "P2q" + "P3P" + "P2q" + "3PPq").pack
pack_softmax_ce = struct.Struct("@2i2q" + 2 * "Pq" + "2Pf" + 2 * "P" + "PPPPPq").pack
_raw_stream = torch._C._cuda_getCurrentRawStream  # (current_stream() builds an object on every call)


def no_tangents(who, *tensors):
  """The sequence operators have gradients, but no forward-mode derivative: a tangent (torch.autograd.forward_ad)
  would be dropped, as the kernels see the primal's memory only."""
  if getattr(forward_ad, "_current_level", 0) < 0:  # (no level is open: spares 3 us a call)
    return
  for x in tensors:
    if x is not None and forward_ad.unpack_dual(x).tangent is not None:
      raise ValueError("%s has no forward-mode derivative" % who)


def launch(name, pack, fields, device):
  """The operator `name` on the current stream of `device`, with `device` the current one (a launch goes to
  it), its arguments packed from `fields` and a workspace from torch's allocator behind them."""
  fn, workspace = _seq_fns[name]
  args = pack(*fields, 0, 0)
  n = workspace(args)
  if n:
    if n < 0:
      check(1)
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    args = pack(*fields, ws.data_ptr(), n)
  index = device.index
  if index == torch.cuda.current_device():
    return check(fn(args, C.c_void_p(_raw_stream(index))))
  with torch.cuda.device(device):
    check(fn(args, C.c_void_p(_raw_stream(index))))
