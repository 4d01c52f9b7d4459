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
is differentiable in ``weight``, as often as asked for, and composes with
``torch.func.vmap``; a derivative of ``embedding_grad`` itself raises.
"""

from __future__ import annotations

import torch

from churten_amd.kernels import _C  # noqa: F401  (registers the ops)
from churten_amd.kernels._replicas import (
    OWN,
    SHARED,
    differentiable,
    register_replica_vmap,
    register_replica_vmap_,
    replica_vmap,
)

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


def _setup(ctx, inputs, output):
    weight, tokens, ctx.scale = inputs
    ctx.num_embeddings = weight.shape[-2]
    ctx.save_for_backward(tokens)


def _backward(ctx, grad):
    tokens, = ctx.saved_tensors
    # A compiled backward pass is not differentiated again.
    once = torch.compiler.is_compiling() or (
        _plain() and not (grad.requires_grad and torch.is_grad_enabled()))
    form = embedding_grad if once else _grad_apply
    return form(grad, tokens, ctx.num_embeddings, ctx.scale), None, None


def _grad_setup(ctx, inputs, output):
    _, tokens, _, ctx.scale = inputs
    ctx.save_for_backward(tokens)


def _grad_backward(ctx, grad):
    # The gradient is linear in the incoming one; its transpose is the lookup.
    tokens, = ctx.saved_tensors
    return embedding(grad, tokens, ctx.scale), None, None, None


_, _grad_apply, _ = differentiable("embedding_grad", _grad_setup, _grad_backward)
_op, _apply, _plain = differentiable("embedding", _setup, _backward)


def embedding(weight: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[n, tokens[n, b]]``; see the module's description."""
    if _plain() and not (weight.requires_grad and torch.is_grad_enabled()):
        return _op(weight, tokens, scale)
    return _apply(weight, tokens, scale)


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
