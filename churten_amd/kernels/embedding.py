"""``churten::embedding`` and its gradient, for every replica at once.

* ``embedding(weight, tokens, scale=1.0)`` -- ``scale * weight[n, tokens[n, b]]``
  as ``(N, B, D)`` in weight's dtype. ``weight`` is ``(N, V, D)``, any view of a
  consolidated buffer among them; ``tokens`` (int64 or int32) is ``(N, B)``, or
  ``(B,)`` where the replicas see the same batch. A token outside ``[0, V)``
  gives a row of zeros and takes no part in the gradient.
* ``embedding_grad(grad, tokens, num_embeddings, scale=1.0)`` -- the ``(N, V,
  D)`` gradient of the table: for each token the rows of ``grad`` at its
  positions, summed in float32 in the order of the positions (the same bits on
  every run), scaled and rounded once.
* ``embedding_grad_(weight_grad, grad, tokens, scale=1.0, accumulate=False)``
  -- the same into a tensor that is there, such as the table's ``(N, V, D)`` view
  of ``State.grads``; with ``accumulate`` added to what it holds (a table that
  another layer shares), where rows that no token names are not touched.

All of them without the replica dimension are one replica's call. ``embedding``
is differentiable in ``weight`` and ``embedding_grad`` in ``grad``, as often as
asked for in reverse mode; all compose with ``torch.func.vmap``.
"""

from __future__ import annotations

import torch

from churten_amd.kernels import _C  # noqa: F401  (registers the ops)
from churten_amd.kernels._replicas import (
    OWN,
    SHARED,
    register_replica_vmap,
    register_replica_vmap_,
    replica_vmap,
)

_op = torch.ops.churten.embedding.default
embedding_grad = torch.ops.churten.embedding_grad
embedding_grad_ = torch.ops.churten.embedding_grad_

__all__ = ["embedding", "embedding_grad", "embedding_grad_"]


@torch.library.register_fake("churten::embedding")
def _embedding_fake(weight, tokens, scale=1.0):
    return weight.new_empty((*weight.shape[:-2], tokens.shape[-1], weight.shape[-1]))


@torch.library.register_fake("churten::embedding_grad")
def _embedding_grad_fake(grad, tokens, num_embeddings, scale=1.0):
    return grad.new_empty((*grad.shape[:-2], num_embeddings, grad.shape[-1]))


@torch.library.register_fake("churten::embedding_grad_")
def _embedding_grad_into_fake(weight_grad, grad, tokens, scale=1.0, accumulate=False):
    return None


def embedding(weight: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[n, tokens[n, b]]``; see the module's description."""
    return _op(weight, tokens, scale)


def _lookups(info, in_dims, weight, tokens, scale=1.0):
    """A table that vmap is not over is looked up once, by the tokens of the whole
    batch: folding the batch into its replicas would repeat it."""
    if in_dims[0] is not None:
        return _replica_lookups(info, in_dims, weight, tokens, scale)
    tokens = tokens.movedim(in_dims[1], -2)
    out = _op(weight, tokens.flatten(-2), scale).unflatten(-2, tokens.shape[-2:])
    return out, out.dim() - 3


_replica_lookups = replica_vmap("embedding", [(OWN, 2), (SHARED, 1)], outputs=1)
torch.library.register_vmap("churten::embedding", _lookups)
register_replica_vmap("embedding_grad", [(OWN, 2), (SHARED, 1)], outputs=1)
register_replica_vmap_("embedding_grad_", [(OWN, 2), (OWN, 2), (SHARED, 1)])
