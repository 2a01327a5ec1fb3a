"""CPU: the sequence and loss operators have no forward-mode derivative, and say so instead of dropping the tangent."""
import pytest
import torch
from torch.autograd import forward_ad

from monolith_amd import attention_ops, embedding_combiners, loss_ops


def _attention(x):
  return attention_ops.ragged_attention(x["query"], x["key"], x["value"], torch.tensor([0, 4, 9]), torch.tensor([0, 2, 6]))


def _pooled(x):
  key = embedding_combiners.Ragged(torch.arange(9), torch.tensor([0, 1, 2, 3, 4, 5, 9]))
  return embedding_combiners.Attention(x["query"].flatten(1)[:, :16], 2).combine(key, x["key"].flatten(1)[:, :16])


def _prefix(x):
  return attention_ops.shared_prefix_attention(x["query"], x["key"], x["value"])


def _prefix_own(x):
  return attention_ops.shared_prefix_attention(torch.zeros(6, 4, 16), torch.zeros(3, 2, 16), None, x["key"], x["value"],
                                               torch.tensor([0, 1, 2, 3, 4, 5, 9]))


def _loss(x):
  return loss_ops.softmax_cross_entropy(x["query"].flatten(1), x["rows"], torch.zeros(6, dtype=torch.int64), x["bias"])


CALLS = [(_attention, ("query", "key", "value")), (_pooled, ("query", "key")), (_prefix, ("query", "key", "value")),
         (_prefix_own, ("key", "value")), (_loss, ("query", "rows", "bias"))]


@pytest.mark.parametrize("call,names", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(call, names, grad):
  shapes = {"query": (6, 4, 16), "key": (9, 2, 16), "value": (9, 2, 16), "rows": (9, 64), "bias": (9,)}
  for name in names:
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
      x = {k: torch.zeros(s) for k, s in shapes.items()}
      x[name] = forward_ad.make_dual(x[name], torch.ones(shapes[name]))
      with pytest.raises(ValueError, match="forward-mode"):
        call(x)
      x = {k: torch.zeros(s, requires_grad=k == name and call in (_attention, _pooled, _loss)) for k, s in shapes.items()}
      with pytest.raises(Exception, match="no CPU fallback"):  # (no tangent: as outside of the level)
        call(x)
