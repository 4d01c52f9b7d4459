"""How the language-model operators meet ``torch.autograd`` and ``torch.func``.

``differentiable`` gives an operator its derivative. Calls that need none go
straight to the operator; the others through a ``torch.autograd.Function``,
which plain autograd and the transforms of ``torch.func`` both take.

``register_replica_vmap`` is the operators' batching rule. They take their
tensors with a leading replica dimension, or all of them without, and some may
be shared by the replicas. So an outer
``torch.func.vmap`` dimension is a replica dimension: over a call without one
it becomes it, over a call that has one both are folded together -- where a
replica's own tensor that vmap is not over is repeated in memory, once for each
of the batch (but for the table of a lookup).
"""

from __future__ import annotations

import torch

__all__ = ["OWN", "SHARED", "HYPER", "TABLE", "differentiable", "register_replica_vmap",
           "register_replica_vmap_", "replica_vmap", "without_derivative"]

OWN = "own"  # every replica has one
SHARED = "shared"  # the replicas may share one
HYPER = "hyper"  # a number for each replica
TABLE = "table"  # one for all


def _fold(t, dim, kind, rank, batch, replicas):
    """``t`` for the folded call: ``rank`` dimensions for one replica, behind
    ``batch * replicas`` of them (``replicas`` is None for a call without the
    dimension) unless it is shared."""
    if dim is not None:
        t = t.movedim(dim, 0)
    if kind is HYPER:
        t = t.reshape((batch if dim is not None else 1, replicas or 1))
        return t.expand(batch, replicas or 1).reshape(-1)
    has_replicas = t.dim() - (dim is not None) > rank
    if dim is None and not has_replicas and kind is SHARED:
        return t
    if dim is None:
        t = t.unsqueeze(0)
    if replicas is None:
        return t.expand(batch, *t.shape[1:])
    if not has_replicas:
        t = t.unsqueeze(1)
    return t.expand(batch, replicas, *t.shape[2:]).flatten(0, 1)


def replica_vmap(name: str, kinds: list[tuple[str, int]], outputs: int):
    """The batching rule of ``churten::name``. ``kinds``: for each tensor argument, in order, what it is to a replica
    and its dimensions for one; the first is a replica's own and shows whether
    the call has the replicas' dimension. ``outputs``: how many tensors the
    operator returns."""
    op = getattr(torch.ops.churten, name)

    def rule(info, in_dims, *args):
        batch, first, dim = info.batch_size, args[0], in_dims[0]
        replicas = None
        if first.dim() - (dim is not None) > kinds[0][1]:
            replicas = (first if dim is None else first.movedim(dim, 0)[0]).shape[0]
        given = list(args)
        for i, (kind, rank) in enumerate(kinds):
            if i >= len(given) or given[i] is None:
                continue
            if kind is TABLE:
                if in_dims[i] is not None:
                    raise RuntimeError(f"churten::{name}: vmap over argument {i}, which every "
                                       "replica shares, is not supported")
                continue
            given[i] = _fold(given[i], in_dims[i], kind, rank, batch, replicas)
        out = op(*given)
        tensors = (out,) if outputs == 1 else out
        if replicas is not None:
            tensors = tuple(t.unflatten(0, (batch, replicas)) for t in tensors)
        return (tensors[0], 0) if outputs == 1 else (tensors, (0,) * outputs)

    return rule


def register_replica_vmap(name: str, kinds: list[tuple[str, int]], outputs: int) -> None:
    torch.library.register_vmap(f"churten::{name}", replica_vmap(name, kinds, outputs))


def register_replica_vmap_(name: str, kinds: list[tuple[str, int]]) -> None:
    """The same for an operator that writes into its first tensor and returns
    nothing."""
    op = getattr(torch.ops.churten, name)

    def rule(info, in_dims, *args):
        batch, dim = info.batch_size, in_dims[0]
        if dim is None:
            raise RuntimeError(f"churten::{name}: its first tensor is written in place, so "
                               "vmap must be over it too")
        out = args[0].movedim(dim, 0)
        replicas = out.shape[1] if out.dim() - 1 > kinds[0][1] else None
        given = list(args)
        for i, (kind, rank) in enumerate(kinds[1:], 1):
            given[i] = _fold(given[i], in_dims[i], kind, rank, batch, replicas)
        if replicas is None:
            op(out, *given[1:])
            return None, None
        try:
            folded = out.view(batch * replicas, *out.shape[2:])
        except RuntimeError:  # no one view: a call for each
            folded = None
        if folded is not None:
            op(folded, *given[1:])
            return None, None
        for b in range(batch):
            own = slice(b * replicas, (b + 1) * replicas)
            op(out[b], *(t[own] if i < len(kinds) and t.dim() > kinds[i][1] else t
                         for i, t in enumerate(given[1:], 1)))
        return None, None

    torch.library.register_vmap(f"churten::{name}", rule)


def differentiable(name: str, setup, backward):
    """``(op, apply, plain)`` of the operator ``churten::name``: itself, the same
    with the derivative that ``backward`` forms from what ``setup(ctx, inputs,
    output)`` left, and whether a call whose tensors ask for no gradient may go
    without."""
    op = getattr(torch.ops.churten, name).default
    function = type(name, (torch.autograd.Function,), {
        "generate_vmap_rule": True,
        "forward": staticmethod(lambda *args: op(*args)),
        "setup_context": staticmethod(setup),
        "backward": staticmethod(backward),
    })
    transforms = torch._C._functorch.peek_interpreter_stack

    def plain() -> bool:
        return transforms() is None and not torch.compiler.is_compiling()

    return op, function.apply, plain


class _WithoutDerivative(torch.autograd.Function):
    generate_vmap_rule = True

    @staticmethod
    def forward(t, what):
        return t.view_as(t)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.what = inputs[1]

    @staticmethod
    def backward(ctx, grad):
        raise NotImplementedError(f"derivative for {ctx.what} is not implemented")


def without_derivative(t, what: str):
    """``t`` for an operator whose backward pass forms no gradient of it: asking
    for one raises instead of finding none."""
    return _WithoutDerivative.apply(t, what) if t is not None and t.requires_grad else t
