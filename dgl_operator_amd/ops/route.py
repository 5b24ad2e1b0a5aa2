"""Rows sorted by group and back: the typed / mixture-of-experts row movement.

``route_rows`` plans it from group ids (relation or node types, a router's
experts): a stable sort of the slots ``(row, choice)`` by group.
``dispatch_rows`` copies every row to its places in the sorted order, where
each group is one contiguous range for ``segment_mm`` or ``segment_reduce``;
``combine_rows`` brings the sorted rows back as a weighted sum per row. Both are
differentiable. On GPU all of it is HIP kernels (csrc/route.hip) that never
synchronise with the host and repeat bit for bit; on CPU it is plain PyTorch.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import backend


class RowRoute(NamedTuple):
    """Where each row goes.

    offsets   int64 [num_groups + 1]: sorted rows offsets[g]..offsets[g+1] are
              group g's, in the order of the rows they come from
    position  int32 [rows, k]: the sorted row of each slot, -1 for a dropped one
    source    int32 [rows * k]: the slot (row * k + choice) of each sorted row,
              -1 behind the last group
    """

    offsets: torch.Tensor
    position: torch.Tensor
    source: torch.Tensor


def route_rows(ids: torch.Tensor, num_groups: int) -> RowRoute:
    """Plan from group ids [rows] or [rows, k] (int32 or int64).

    An id outside [0, num_groups) drops its slot: it is copied nowhere and adds
    nothing when the rows come back, as a padded row should. On GPU num_groups
    is at most 16384.
    """
    assert ids.dim() in (1, 2), "route_rows: ids must be [rows] or [rows, k]"
    assert ids.dtype in (torch.int32, torch.int64), \
        "route_rows: int32 or int64 ids expected"
    assert num_groups >= 1, "route_rows: num_groups must be positive"
    if ids.dim() == 1:
        ids = ids.unsqueeze(1)
    if ids.is_cuda:
        ext = backend.ext_for(ids)
        return RowRoute(*ext.route_rows(ids, num_groups))
    flat = ids.reshape(-1).long()
    kept = (flat >= 0) & (flat < num_groups)
    key = torch.where(kept, flat, num_groups)
    order = torch.argsort(key, stable=True)
    offsets = torch.zeros(num_groups + 1, dtype=torch.int64)
    offsets[1:] = torch.cumsum(
        torch.bincount(key, minlength=num_groups + 1)[:num_groups], 0)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel())
    return RowRoute(
        offsets,
        torch.where(kept, place, -1).view(ids.shape).int(),
        torch.where(kept[order], order, -1).int(),
    )


def _dispatch_ref(x: torch.Tensor, position: torch.Tensor) -> torch.Tensor:
    k = position.shape[1]
    flat = position.reshape(-1).long()
    kept = (flat >= 0).nonzero()[:, 0]
    out = x.new_zeros((flat.numel(), x.shape[1]))
    out[flat[kept]] = x[kept // k] if k else x[:0]
    return out


def _taken_ref(y: torch.Tensor, position: torch.Tensor) -> torch.Tensor:
    """y's rows by slot, [rows, k, D], zero where dropped, in >= 32 bits."""
    rows, k = position.shape
    flat = position.reshape(-1).long()
    kept = (flat >= 0).nonzero()[:, 0]
    acc = y.dtype if y.dtype == torch.float64 else torch.float32
    out = torch.zeros((rows * k, y.shape[1]), dtype=acc)
    out[kept] = y[flat[kept]].to(acc)
    return out.view(rows, k, y.shape[1])


def _combine_ref(y, position, weights):
    taken = _taken_ref(y, position)
    if weights is not None:
        taken = taken * weights.to(taken.dtype).unsqueeze(-1)
    return taken.sum(1).to(y.dtype)


class _DispatchRows(torch.autograd.Function):
    """CPU path; the GPU's is csrc/autograd.cpp."""

    @staticmethod
    def forward(ctx, x, position):
        ctx.save_for_backward(position)
        return _dispatch_ref(x, position)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        (position,) = ctx.saved_tensors
        return _combine_ref(grad_out, position, None), None


class _CombineRows(torch.autograd.Function):
    """CPU path; the GPU's is csrc/autograd.cpp."""

    @staticmethod
    def forward(ctx, y, weights, position):
        ctx.save_for_backward(y, weights, position)
        return _combine_ref(y, position, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        y, w, position = ctx.saved_tensors
        dy = dw = None
        rows, k = position.shape
        if ctx.needs_input_grad[0]:
            g = grad_out.unsqueeze(1).expand(rows, k, grad_out.shape[1])
            if w is not None:
                g = (g.to(torch.promote_types(g.dtype, torch.float32))
                     * w.unsqueeze(-1)).to(grad_out.dtype)
            flat = position.reshape(-1).long()
            kept = (flat >= 0).nonzero()[:, 0]
            dy = grad_out.new_zeros((rows * k, grad_out.shape[1]))
            dy[flat[kept]] = g.reshape(rows * k, -1)[kept]
        if ctx.needs_input_grad[1]:
            taken = _taken_ref(y, position)
            dw = (taken * grad_out.to(taken.dtype).unsqueeze(1)).sum(-1)
            dw = dw.to(w.dtype)
        return dy, dw, None


def dispatch_rows(route: RowRoute, x: torch.Tensor) -> torch.Tensor:
    """x [rows, ...] -> sorted rows [rows * k, ...]: row ``route.position[t, j]``
    is x[t]; rows behind the last group are zero. Its gradient sums the copies
    of each row. On GPU a row has fewer than 2^30 elements."""
    rows, k = route.position.shape
    assert x.dim() >= 2 and x.shape[0] == rows, \
        f"dispatch_rows: [{rows}, ...] rows expected, got {tuple(x.shape)}"
    assert x.device == route.position.device, \
        "dispatch_rows: rows and plan are on different devices"
    assert x.is_floating_point(), "dispatch_rows: floating point rows expected"
    if x.is_cuda:
        ext = backend.ext_for(x)
        out = ext.dispatch_rows(_flat(x), route.position, route.offsets)
    else:
        out = _DispatchRows.apply(_flat(x), route.position)
    if x.dim() == 2:
        return out
    return out.view((rows * k,) + x.shape[1:])


def combine_rows(
    route: RowRoute, y: torch.Tensor, weights: Optional[torch.Tensor] = None
) -> torch.Tensor:
    """Sorted rows y [rows * k, ...] -> [rows, ...]:
    out[t] = sum_j weights[t, j] * y[route.position[t, j]], dropped slots adding
    nothing. weights is [rows, k] (any float type; all ones when None; [rows]
    will do for k = 1). Sums are in 32 bits, rounded once, on GPU with the weights
    in 32 bits too; gradients reach y and weights. On GPU a row has fewer than
    2^30 elements."""
    rows, k = route.position.shape
    assert y.dim() >= 2 and y.shape[0] == rows * k, \
        f"combine_rows: [{rows * k}, ...] rows expected, got {tuple(y.shape)}"
    assert y.device == route.position.device, \
        "combine_rows: rows and plan are on different devices"
    assert y.is_floating_point(), "combine_rows: floating point rows expected"
    if weights is not None:
        if k == 1 and weights.dim() == 1:
            weights = weights.unsqueeze(1)
        assert weights.shape == route.position.shape, \
            f"combine_rows: weights must be [{rows}, {k}]"
        assert weights.device == y.device and weights.is_floating_point(), \
            "combine_rows: floating point weights on the rows' device expected"
    if y.is_cuda:
        ext = backend.ext_for(y)
        out = ext.combine_rows(_flat(y), weights, route.position, route.offsets)
    else:
        out = _CombineRows.apply(_flat(y), weights, route.position)
    if y.dim() == 2:
        return out
    return out.view((rows,) + y.shape[1:])


def _flat(x: torch.Tensor) -> torch.Tensor:
    if x.dim() == 2:
        return x
    width = 1
    for d in x.shape[1:]:
        width *= d
    return x.reshape(x.shape[0], width)
