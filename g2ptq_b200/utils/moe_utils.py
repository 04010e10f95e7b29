"""Expert routing for MoE blocks: tokens to experts and back.

The reference's routed expert forward (``_forward_with_split_experts``,
utils/models/mixins.py:233-259) indexes each hit expert's tokens, runs the
expert on them and adds the weighted results back, so that the expert
linears' hooks (``add_batch``, the refresh step's caches) see routed tokens
only.  Here the pairs are sorted by expert once (``route``), the rows are copied
into that order in one pass (``dispatch``) and brought back weighted in one
pass (``combine``), both differentiable; ``routed_experts_forward`` is that
forward.
"""

import collections

import torch

from .. import ops

#: ``order [T k]``, ``position [T, k]`` and ``offsets [E + 1]`` of ``ops.route``.
Routing = collections.namedtuple("Routing", ("order", "position", "offsets"))


def route(experts, num_experts):
    """The ``Routing`` of the expert ids ``experts [T, k]``.  Ids outside of
    ``[0, num_experts)`` (experts of another process, dropped slots) take part
    in nothing: their rows are zero and add nothing."""
    return Routing(*ops.route(experts.contiguous(), num_experts))


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position):
        ctx.save_for_backward(position)
        return ops.dispatch_rows(x, position)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (position,) = ctx.saved_tensors
        return ops.combine_rows(_rows(grad), position), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, position, weights):
        ctx.save_for_backward(y if ctx.needs_input_grad[2] else None, position, weights)
        return ops.combine_rows(y, position, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        y, position, weights = ctx.saved_tensors
        grad = _rows(grad)
        need_y, _, need_w = ctx.needs_input_grad
        if weights is None:
            return (ops.dispatch_rows(grad, position) if need_y else None), None, None
        gy, gw = ops.combine_rows_backward(grad, y, position, weights, need_y, need_w)
        return gy, None, gw


def _rows(t):
    """``t`` with unit column stride and rows that do not overlap (a gradient
    that autograd broadcast can have stride zero)."""
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        return t.contiguous()
    return t


def _records(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def dispatch(x, routing):
    """``x [T, C]`` in expert order: ``[T k, C]``, row ``r`` the token of pair
    ``routing.order[r]``; rows of pairs without an expert are zero."""
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32) and _records(x):
        raise TypeError(f"unsupported dtype {x.dtype}")
    x = _rows(x) if x.dim() == 2 else x
    if _records(x):
        return _Dispatch.apply(x, routing.position)
    return ops.dispatch_rows(x, routing.position)


def combine(y, routing, weights=None):
    """Expert rows ``y [T k, C]`` back in token order, weighted by ``weights
    [T, k]`` (None: ones) and summed over the slots: ``[T, C]``."""
    y = _rows(y) if y.dim() == 2 else y
    weights = None if weights is None else weights.contiguous()
    if _records(y, weights):
        return _Combine.apply(y, routing.position, weights)
    return ops.combine_rows(y, routing.position, weights)


def routed_experts_forward(experts, hidden, top_experts, top_weights):
    """The reference's routed expert forward: ``experts[e]`` (a callable, an
    expert's MLP) runs on its routed tokens of ``hidden [T, C]`` only -- experts
    that no token chose are not called -- and the results are added back with
    the router's weights ``top_weights [T, k]``.  Differentiable; reads the
    expert's row counts back to the host once, as the reference's loop over hit
    experts does."""
    routing = route(top_experts, len(experts))
    rows = dispatch(hidden, routing)
    cut = routing.offsets.tolist()
    parts = [experts[e](rows[a:b]) for e, (a, b) in enumerate(zip(cut, cut[1:])) if b > a]
    if not parts:  # zeros, and zero gradients
        return combine(rows, routing, top_weights)
    tail = rows.shape[0] - cut[-1]
    if tail:
        parts.append(parts[0].new_zeros(tail, parts[0].shape[1]))
    return combine(torch.cat(parts), routing, top_weights)
