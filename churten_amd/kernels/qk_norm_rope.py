"""``churten::qk_norm_rope``: the norm of each query and key head and its
rotation by position, in one pass over the heads, and its backward pass.

``qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps=1e-6,
interleaved=False) -> (q, k)``

* ``q`` ``(N, M, Hq, D)`` and ``k`` ``(N, M, Hk, D)``: the heads of each
  replica's M tokens, any strides (slices of one fused projection).
* ``q_weight``, ``k_weight`` ``(N, D)``: learned weights, in q's dtype. Each head
  ``x`` becomes ``x * rsqrt(mean(x^2) + eps) * weight``.
* ``cos``, ``sin`` ``(P, r)`` float32: the angles of ``r <= D / 2`` pairs at P
  positions; the first ``2 r`` elements rotate, as the pairs ``(j, j + r)``, or
  with ``interleaved`` ``(2 j, 2 j + 1)``; the others pass.
* ``positions`` ``(N, M)`` or ``(M,)``, int64 or int32: rows of the tables. A
  position outside ``[0, P)`` does not rotate.

``qk_norm_rope_grad(grad_q, grad_k, q, k, ...)`` gives the gradients of ``q``,
``k``, ``q_weight`` and ``k_weight`` from those of the results; it forms the norms
anew from ``q`` and ``k``. Arithmetic is float32, each result rounded once.

All tensors without the replica dimension are one replica's call. The operator
is differentiable once in q, k and the weights and composes with
``torch.func.vmap``; asking for a second derivative, or for one in the angles, raises.
"""

from __future__ import annotations

import torch

from churten_amd.kernels import _C  # noqa: F401  (registers the ops)
from churten_amd.kernels._replicas import (
    OWN,
    SHARED,
    TABLE,
    differentiable,
    register_replica_vmap,
    without_derivative,
)

qk_norm_rope_grad = torch.ops.churten.qk_norm_rope_grad

__all__ = ["qk_norm_rope", "qk_norm_rope_grad"]


@torch.library.register_fake("churten::qk_norm_rope")
def _qk_norm_rope_fake(q, k, q_weight, k_weight, cos, sin, positions, eps=1e-6,
                       interleaved=False):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.register_fake("churten::qk_norm_rope_grad")
def _qk_norm_rope_grad_fake(grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, positions,
                            eps=1e-6, interleaved=False):
    return (q.new_empty(q.shape), k.new_empty(k.shape), q_weight.new_empty(q_weight.shape),
            k_weight.new_empty(k_weight.shape))


def _setup(ctx, inputs, output):
    *tensors, ctx.eps, ctx.interleaved = inputs
    ctx.save_for_backward(*tensors)


def _backward(ctx, grad_q, grad_k):
    q, k = ctx.saved_tensors[:2]
    grad_q = torch.zeros_like(q) if grad_q is None else grad_q
    grad_k = torch.zeros_like(k) if grad_k is None else grad_k
    grads = qk_norm_rope_grad(grad_q, grad_k, *ctx.saved_tensors, ctx.eps, ctx.interleaved)
    return (*grads, None, None, None, None, None)


_op, _apply, _plain = differentiable("qk_norm_rope", _setup, _backward)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
                 k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 positions: torch.Tensor, eps: float = 1e-6,
                 interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """The normed and rotated ``(q, k)``; see the module's description."""
    tracked = (q.requires_grad or k.requires_grad or q_weight.requires_grad
               or k_weight.requires_grad) and torch.is_grad_enabled()
    if _plain() and not tracked:
        return _op(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    return _apply(q, k, q_weight, k_weight, without_derivative(cos, "qk_norm_rope in cos"),
                  without_derivative(sin, "qk_norm_rope in sin"), positions, eps, interleaved)


_INPUTS = [(OWN, 3), (OWN, 3), (OWN, 1), (OWN, 1), (TABLE, 2), (TABLE, 2), (SHARED, 1)]
register_replica_vmap("qk_norm_rope", _INPUTS, outputs=2)
register_replica_vmap("qk_norm_rope_grad", [(OWN, 3), (OWN, 3), *_INPUTS], outputs=4)
