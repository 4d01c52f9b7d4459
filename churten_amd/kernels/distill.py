"""``churten::distill_loss``: distillation from a teacher's top logits, and its
gradient, for every replica at once.

``distill_loss(logits, teacher_logits, teacher_index, temperature, weight=None,
labels=None, hard=None) -> (N, B) float32``

For each row, with x the student's V logits, z the teacher's K top logits at
the indices i, t the replica's temperature and h its share of hard labels::

    p    = softmax(z / t) over the row's present entries
    loss = weight * ((1 - h) * t^2 * sum_k p_k (log p_k - log softmax(x / t)[i_k])
                     + h * -log softmax(x)[label])

* ``logits`` ``(N, B, V)`` in float32, float16 or bfloat16; rows may be strided.
* ``teacher_logits``, ``teacher_index`` ``(N, B, K)``, or ``(B, K)`` for one teacher
  of all replicas; K <= 1024. An entry whose index lies outside ``[0, V)`` or
  whose logit is -infinity is absent; a row without entries has only its hard
  part. Entries that name one index add up. No gradient flows to the teacher.
* ``temperature`` ``(N,)``, positive, and ``hard`` ``(N,)``: per-replica
  hyperparameters.
* ``weight`` ``(N, B)`` or ``(B,)``: a row of weight 0 (padding, a frozen replica)
  is not read, whatever its logits hold; its loss and gradient are 0.
* ``labels`` ``(N, B)`` or ``(B,)``, given together with ``hard``: a label outside
  ``[0, V)`` has no hard part. A replica with h = 0 has no hard part and one with
  h = 1 none from the teacher, also where those would be infinite.

``distill_loss_grad`` (same arguments) returns the loss and the gradient of its
sum over all rows in the logits, in one pass over them: a training step that
has no other use of autograd's graph takes this one. ``distill_loss`` is
differentiable once in ``logits`` and composes with ``torch.func.vmap``; asking for a
second derivative, or for one in ``temperature``, ``weight`` or ``hard``, raises.
"""

from __future__ import annotations

import torch

from churten_amd.kernels import _C  # noqa: F401  (registers the ops)
from churten_amd.kernels._replicas import (
    HYPER,
    OWN,
    SHARED,
    differentiable,
    register_replica_vmap,
    without_derivative,
)

distill_loss_grad = torch.ops.churten.distill_loss_grad

__all__ = ["distill_loss", "distill_loss_grad"]


@torch.library.register_fake("churten::distill_loss")
def _distill_loss_fake(logits, teacher_logits, teacher_index, temperature, weight=None,
                       labels=None, hard=None):
    return logits.new_empty(logits.shape[:-1], dtype=torch.float32)


@torch.library.register_fake("churten::distill_loss_grad")
def _distill_loss_grad_fake(logits, teacher_logits, teacher_index, temperature, weight=None,
                            labels=None, hard=None):
    return (logits.new_empty(logits.shape[:-1], dtype=torch.float32),
            logits.new_empty(logits.shape))


def _setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _backward(ctx, grad):
    logits, z, index, temperature, weight, labels, hard = ctx.saved_tensors
    # The loss is linear in its row's weight, so the weight carries the
    # incoming gradient: rows that receive none are not read.
    weight = grad if weight is None else grad * weight
    _, grad_logits = distill_loss_grad(logits, z, index, temperature, weight, labels, hard)
    return grad_logits, None, None, None, None, None, None


_op, _apply, _plain = differentiable("distill_loss", _setup, _backward)


def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor,
                 teacher_index: torch.Tensor, temperature: torch.Tensor,
                 weight: torch.Tensor | None = None, labels: torch.Tensor | None = None,
                 hard: torch.Tensor | None = None) -> torch.Tensor:
    """The rows' losses; see the module's description."""
    if teacher_logits.requires_grad:
        teacher_logits = teacher_logits.detach()
    if _plain() and not (logits.requires_grad and torch.is_grad_enabled()):
        return _op(logits, teacher_logits, teacher_index, temperature, weight, labels, hard)
    return _apply(logits, teacher_logits, teacher_index,
                  without_derivative(temperature, "distill_loss in temperature"),
                  without_derivative(weight, "distill_loss in weight"), labels,
                  without_derivative(hard, "distill_loss in hard"))


_INPUTS = [(OWN, 2), (SHARED, 2), (SHARED, 2), (HYPER, 0), (SHARED, 1), (SHARED, 1), (HYPER, 0)]
register_replica_vmap("distill_loss", _INPUTS, outputs=1)
register_replica_vmap("distill_loss_grad", _INPUTS, outputs=2)
