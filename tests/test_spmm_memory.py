"""The CPU spmm sums in 64 bits without holding all messages."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from dgl_operator_amd.ops import spmm
from dgl_operator_amd.ops.spmm import spmm_raw


class Largest(TorchDispatchMode):
    """Elements of the largest floating point result that has a row an edge."""

    def __init__(self):
        super().__init__()
        self.most = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if isinstance(out, torch.Tensor) and out.is_floating_point():
            self.most = max(self.most, out.numel())
        return out


def graph(rows, edges, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ends = torch.randint(0, edges + 1, (rows - 1,), generator=gen).sort().values
    indptr = torch.cat((torch.tensor([0]), ends, torch.tensor([edges])))
    return indptr, torch.randint(0, rows, (edges,), generator=gen)


@pytest.mark.parametrize("shape", [(7,), (3, 5), (1, 4)])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("mean", [False, True])
@pytest.mark.parametrize("elements", [1, 100, 1 << 20])
def test_sums_do_not_depend_on_the_stretches(monkeypatch, shape, weighted, mean,
                                             elements):
    rows, edges = 40, 1000
    indptr, indices = graph(rows, edges)
    feat = torch.randn(rows, *shape)
    weight = torch.rand((edges,) + shape[:-1]) if weighted else None
    monkeypatch.setattr(spmm, "_REF_ELEMENTS", elements)
    got = spmm_raw(indptr, indices, feat, weight, mean)
    ref = torch.zeros(rows, *shape, dtype=torch.float64)
    for v in range(rows):
        for e in range(int(indptr[v]), int(indptr[v + 1])):
            m = feat[indices[e]]
            ref[v] += m if weight is None else m * weight[e].unsqueeze(-1)
    if mean:
        deg = (indptr[1:] - indptr[:-1]).clamp(min=1).double()
        ref /= deg.view(-1, *[1] * len(shape))
    assert torch.equal(got, ref.float())


def test_messages_are_not_held_at_once():
    rows, edges, width = 50, 100_000, 64
    indptr, indices = graph(rows, edges)
    feat = torch.randn(rows, width)
    with Largest() as seen:
        spmm_raw(indptr, indices, feat, torch.rand(edges), True)
    assert seen.most <= 1 << 20 < edges * width


def test_no_edges_and_no_features():
    indptr = torch.zeros(4, dtype=torch.int64)
    none = torch.empty(0, dtype=torch.int64)
    assert torch.equal(spmm_raw(indptr, none, torch.ones(3, 2)),
                       torch.zeros(3, 2))
    indptr, indices = graph(3, 9)
    assert spmm_raw(indptr, indices, torch.ones(3, 0)).shape == (3, 0)
