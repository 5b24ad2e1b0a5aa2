"""Product of each group of rows with its own weight (typed / expert product).

``segment_mm(offsets, x, weight)`` is y[r] = x[r] @ weight[g] for the rows
offsets[g]..offsets[g+1] of every group g, the layout ``route_rows`` and
``segment_reduce`` use: relation-typed projections, heterogeneous layers, a
mixture's experts. GPU: hand-written MFMA kernels (csrc/segment_mm.hip), one
launch whatever the groups' sizes, no host synchronisation; CPU: plain PyTorch.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import backend


def _bounds(offsets: torch.Tensor, rows: int):
    ends = offsets.clamp(0, rows).tolist()
    return [(g, a, b) for g, (a, b) in enumerate(zip(ends[:-1], ends[1:]))
            if a < b]


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


def _segment_mm_ref(offsets, x, weight):
    y = x.new_zeros((x.shape[0], weight.shape[2]))
    for g, a, b in _bounds(offsets, x.shape[0]):
        y[a:b] = (_wide(x[a:b]) @ _wide(weight[g])).to(y.dtype)
    return y


class _SegmentMM(torch.autograd.Function):
    """CPU path; the GPU's is csrc/autograd.cpp."""

    @staticmethod
    def forward(ctx, offsets, x, weight):
        ctx.save_for_backward(offsets, x, weight)
        return _segment_mm_ref(offsets, x, weight)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        offsets, x, weight = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[1]:
            dx = _segment_mm_ref(offsets, grad_out, weight.transpose(1, 2))
        if ctx.needs_input_grad[2]:
            dw = x.new_zeros((offsets.numel() - 1, x.shape[1],
                              grad_out.shape[1]))
            for g, a, b in _bounds(offsets, x.shape[0]):
                dw[g] = (_wide(x[a:b]).t() @ _wide(grad_out[a:b])).to(dw.dtype)
        return None, dx, dw


def segment_mm(offsets: torch.Tensor, x: torch.Tensor,
               weight: torch.Tensor) -> torch.Tensor:
    """y[r] = x[r] @ weight[g] for offsets[g] <= r < offsets[g+1].

    offsets  int64 [groups + 1], not falling, within [0, rows]
    x        [rows, K] fp32, bf16 or fp16 (fp64 on CPU too), any row stride
    weight   [groups, K, N] of the same type, any strides (a transposed view of
             [groups, N, K] is read in place)

    Groups may be empty; rows of no group give zeros. Products accumulate in
    fp32 and are rounded once. Gradients reach x and weight. On GPU rows, K and N
    are below 2^30, and what would take more blocks than one launch holds (16
    million tiles of at least 32 x 64) is refused.
    """
    assert offsets.dim() == 1 and offsets.dtype == torch.int64, \
        "segment_mm: int64 offsets [groups + 1] expected"
    assert x.dim() == 2 and weight.dim() == 3, \
        "segment_mm: x [rows, K] and weight [groups, K, N] expected"
    assert weight.shape[0] >= 1 and offsets.numel() == weight.shape[0] + 1, \
        f"segment_mm: {weight.shape[0]} weights need {weight.shape[0] + 1} offsets"
    assert x.shape[1] == weight.shape[1], \
        f"segment_mm: rows of {x.shape[1]} by weights of {weight.shape[1]}"
    assert x.dtype == weight.dtype and x.is_floating_point(), \
        "segment_mm: x and weight must share a floating point type"
    assert x.device == weight.device == offsets.device, \
        "segment_mm: all tensors must be on one device"
    offsets = offsets.contiguous()
    if x.is_cuda:
        return backend.ext_for(x).segment_mm(offsets, x, weight)
    return _SegmentMM.apply(offsets, x, weight)
