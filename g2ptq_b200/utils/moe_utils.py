"""Expert routing for MoE blocks: tokens to experts and back.

The reference's routed expert forward (``_forward_with_split_experts``,
utils/models/mixins.py:233-259) indexes each hit expert's tokens, runs the
expert on them and adds the weighted results back, so that the expert
linears' hooks (``add_batch``, the refresh step's caches) see routed tokens
only.  Here the pairs are sorted by expert once (``route``), the rows are copied
into that order in one pass (``dispatch``) and brought back weighted in one
pass (``combine``), both differentiable (once, backward; forward-mode tangents are
refused); ``routed_experts_forward`` is that forward.
"""

import collections

import torch

from .. import _lib, ops

#: ``order [T k]``, ``position [T, k]`` and ``offsets [E + 1]`` of ``ops.route``.
Routing = collections.namedtuple("Routing", ("order", "position", "offsets"))


def route(experts, num_experts):
    """The ``Routing`` of the expert ids ``experts [T, k]``.  Ids outside of
    ``[0, num_experts)`` (experts of another process, dropped slots) take part
    in nothing: their rows are zero and add nothing."""
    return Routing(*ops.route(experts.contiguous(), num_experts))


def dispatch(x, routing):
    """``x [T, C]`` in expert order: ``[T k, C]``, row ``r`` the token of pair
    ``routing.order[r]``; rows of pairs without an expert are zero."""
    return _lib.binding().dispatch(x, routing.position)


def combine(y, routing, weights=None):
    """Expert rows ``y [T k, C]`` back in token order, weighted by ``weights
    [T, k]`` (None: ones) and summed over the slots: ``[T, C]``."""
    return _lib.binding().combine(y, routing.position, weights)


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
