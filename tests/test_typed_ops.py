"""Rows sorted by group and back, the typed product and log probabilities: the
CPU path, the refusals, and the operators run together."""
import math

import pytest
import torch

import typed_oracle as oracle
from dgl_operator_amd import ops


@pytest.mark.parametrize("rows,k,groups", [
    (0, 1, 1), (1, 1, 1), (1, 3, 5), (7, 2, 3), (64, 1, 1), (130, 4, 17),
])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_route_rows(rows, k, groups, dtype):
    ids = torch.randint(-2, groups + 2, (rows, k), dtype=dtype)
    offsets, position, source = oracle.route(ids, groups)
    got = ops.route_rows(ids, groups)
    assert torch.equal(got.offsets, offsets)
    assert torch.equal(got.position, position.view(rows, k))
    assert torch.equal(got.source, source)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_dispatch_combine(dtype):
    ids = torch.tensor([[0, 2], [2, 2], [-1, 0], [5, -1], [1, 1]])
    route = ops.route_rows(ids, 4)
    x = torch.randn(5, 2, 3, dtype=dtype)
    xs = ops.dispatch_rows(route, x)
    assert xs.shape == (10, 2, 3)
    assert torch.equal(xs.view(10, 6), oracle.dispatch(x.view(5, 6), route.position))
    y, w = torch.randn(10, 6, dtype=dtype), torch.rand(5, 2)
    for weights in (None, w):
        ref, tol = oracle.combine(y, route.position, weights)
        out = ops.combine_rows(route, y, weights)
        assert out.dtype == dtype
        assert ((out.double() - ref).abs() <= tol).all()
    # the row that was dropped twice has nothing
    assert not ops.combine_rows(route, y, w)[3].any()


def test_dispatch_combine_gradients():
    ids = torch.tensor([[0, 2], [2, 2], [-1, 0], [5, -1], [1, 1]])
    route = ops.route_rows(ids, 4)
    x = torch.randn(5, 3, dtype=torch.float64, requires_grad=True)
    y = torch.randn(10, 3, dtype=torch.float64, requires_grad=True)
    w = torch.rand(5, 2, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a: ops.dispatch_rows(route, a), x)
    assert torch.autograd.gradcheck(
        lambda a, b: ops.combine_rows(route, a, b), (y, w))
    assert torch.autograd.gradcheck(lambda a: ops.combine_rows(route, a), y)


def test_route_refusals():
    with pytest.raises(AssertionError):
        ops.route_rows(torch.zeros(2, 2, 2, dtype=torch.int64), 3)
    with pytest.raises(AssertionError):
        ops.route_rows(torch.zeros(4), 3)
    with pytest.raises(AssertionError):
        ops.route_rows(torch.zeros(4, dtype=torch.int64), 0)
    route = ops.route_rows(torch.zeros(4, 2, dtype=torch.int64), 3)
    for bad in (torch.zeros(3, 2), torch.zeros(4), torch.zeros(4, 2).long()):
        with pytest.raises(AssertionError):
            ops.dispatch_rows(route, bad)
    for y, w in ((torch.zeros(4, 2), None),
                 (torch.zeros(8, 2), torch.zeros(4)),
                 (torch.zeros(8, 2), torch.zeros(4, 2).long())):
        with pytest.raises(AssertionError):
            ops.combine_rows(route, y, w)


@pytest.mark.parametrize("sizes", [[3, 0, 2], [0, 0], [1], [5, 1, 0, 4]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64])
def test_segment_mm(sizes, dtype):
    # two rows before the first group, one behind the last
    offsets = torch.tensor([2] + sizes).cumsum(0)
    rows = int(offsets[-1]) + 1
    x = torch.randn(rows, 5, dtype=dtype, requires_grad=True)
    w = torch.randn(len(sizes), 7, 5, dtype=dtype).transpose(1, 2)
    w.requires_grad_()
    g = torch.randn(rows, 7, dtype=dtype)
    y = ops.segment_mm(offsets, x, w)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    for got, (ref, tol) in (
        (y, oracle.segment_mm(offsets, x, w)),
        (dx, oracle.segment_mm(offsets, g, w.transpose(1, 2))),
        (dw, oracle.segment_wgrad(offsets, x, g)),
    ):
        assert got.dtype == dtype
        assert ((got.double() - ref).abs() <= tol).all()
    assert not y[:2].any() and not y[-1].any() and not dx[:2].any()


def test_segment_mm_gradcheck():
    offsets = torch.tensor([0, 2, 2, 5])
    x = torch.randn(6, 3, dtype=torch.float64, requires_grad=True)
    w = torch.randn(3, 3, 4, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(
        lambda a, b: ops.segment_mm(offsets, a, b), (x, w))


def test_segment_mm_refusals():
    o, x, w = torch.tensor([0, 2, 4]), torch.zeros(4, 3), torch.zeros(2, 3, 5)
    for bad in ((o[:2], x, w), (o.int(), x, w), (o, x[:, :2], w),
                (o, x.half(), w), (o, x[0], w), (o, x, w[0]),
                (o, x.long(), w.long())):
        with pytest.raises(AssertionError):
            ops.segment_mm(*bad)


ROWS = {
    "plain": [0.5, -1.0, 2.0, 0.0, -3.0],
    "ties": [1.0, 1.0, -0.0, 0.0, 1.0],
    "masked": [-math.inf, 1.0, -math.inf, 0.0, -math.inf],
    "one left": [-math.inf, -math.inf, -4.0, -math.inf, -math.inf],
    "none left": [-math.inf] * 5,
    "lowest": [torch.finfo(torch.float32).min] * 4 + [0.0],
    "all lowest": [torch.finfo(torch.float32).min] * 5,
    "far": [1e6, 1e6 + 1, 1e6 - 2, 1e6, 1e6 + 0.5],
}


def check_log_probs(device, z, target, k, ignore=-100, grads=True):
    """Forward and backward against the oracle, at derived bounds."""
    rows, C = z.shape
    zc = z.cpu()
    lp, ent, top, index, logp = oracle.log_probs(zc, target, k, ignore)
    zd = z.detach().to(device).requires_grad_(grads)
    td = None if target is None else target.to(device)
    got = ops.log_probs(zd, td, top_k=k, ignore_index=ignore)
    assert torch.equal(got.top_index.cpu(), index)
    u, s_err = oracle.U, oracle.log_s_error(zc)
    spread = (zc.double().amax(1, keepdim=True) - zc.double())
    spread = torch.where(torch.isfinite(spread), spread, 0.0)

    def near(a, b, tol):
        a = a.detach().double().cpu()
        same = (a == b) | (torch.isnan(a) & torch.isnan(b))
        assert (same | ((a - b).abs() <= tol)).all(), \
            ((a - b).abs() - tol).nan_to_num(0).max()

    # (z - m) rounded, log s, their difference rounded
    tol = u * (2 * logp.abs() + spread) + s_err
    tol = torch.where(torch.isfinite(tol), tol, 0.0)
    if target is None:
        assert got.log_prob is None
    else:
        near(got.log_prob, lp, tol.gather(
            1, target.clamp(0, C - 1)[:, None])[:, 0])
    near(got.top_log_prob, top, tol.gather(1, index))
    # a / s: sums of |z - m| e^(z - m), at most log C + 1 of them, each with
    # the steps of s and the roundings of (z - m) and of the product
    p = logp.exp().nan_to_num(0)
    mean = (p * spread).sum(1)
    ent_tol = 2 * s_err * (mean + 1) + 4 * u * (p * spread * spread).sum(1) \
        + 2 * u * (ent.abs() + mean)
    near(got.entropy, ent, ent_tol)
    if not grads:
        return
    g = [torch.randn(rows), torch.randn(rows), torch.randn(rows, k)]
    used = [None if target is None else g[0], g[1], g[2] if k else None]
    outs = [o for o, v in zip(got[:3], used) if v is not None]
    (dz,) = torch.autograd.grad(
        outs, zd, [v.to(device) for v in used if v is not None])
    assert dz.dtype == z.dtype and dz.shape == z.shape
    ref = oracle.log_probs_grad(zc, target, index, logp, ent, *used, ignore)
    # p is off by its logarithm's error; every term is rounded a few times
    size = sum(v.abs().double().view(rows, -1).sum(1)
               for v in (used[0], used[2]) if v is not None)
    size = size + torch.zeros(rows)
    fl = logp.abs() + ent.abs()[:, None]
    fl = torch.where(torch.isfinite(fl), fl, 0.0)
    rel = tol + 8 * u
    gtol = p * (size[:, None] * (2 * rel + (k + 4) * u)
                + g[1].abs().double()[:, None]
                * (fl * (2 * rel + 8 * u) + tol + ent_tol[:, None]))
    own = torch.zeros_like(ref)
    if used[0] is not None:
        own.scatter_add_(1, target.clamp(0, C - 1)[:, None],
                         used[0].abs().double()[:, None])
    if used[2] is not None:
        own.scatter_add_(1, index, used[2].abs().double())
    gtol = gtol + (k + 4) * u * own
    gtol = torch.where(torch.isfinite(gtol), gtol, 0.0)
    near(dz, ref, gtol + oracle.half(z.dtype) * (ref.abs() + gtol)
         + oracle.tiny(z.dtype))


@pytest.mark.parametrize("name", sorted(ROWS))
def test_log_probs_rows(name):
    z = torch.tensor([ROWS[name]] * 3)
    check_log_probs("cpu", z, torch.tensor([0, 2, 4]), 5)


@pytest.mark.parametrize("C", [1, 2, 47, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_log_probs_sizes(C, dtype):
    z = (torch.randn(6, C) * 3).to(dtype)
    check_log_probs("cpu", z, torch.randint(0, C, (6,)), min(C, 5))
    check_log_probs("cpu", z, None, 0)


def test_log_probs_targets():
    z = torch.randn(4, 6)
    check_log_probs("cpu", z, torch.tensor([1, -100, 6, -1]), 2)
    check_log_probs("cpu", z, torch.tensor([1, 5, 5, 0]), 0, ignore=5)


def test_log_probs_not_finite():
    z = torch.tensor([[0.0, math.nan, 2.0], [math.inf, 0.0, 1.0]])
    a = ops.log_probs(z, torch.tensor([0, 1]), top_k=2)
    assert a.log_prob.isnan().all() and a.entropy.isnan().all()
    assert a.top_log_prob.isnan().all()
    assert a.top_index.tolist() == [[1, 2], [0, 2]]


def test_log_probs_shapes_and_gradcheck():
    z = torch.randn(2, 3, 5, dtype=torch.float64, requires_grad=True)
    t = torch.randint(0, 5, (2, 3))
    a = ops.log_probs(z, t, top_k=2)
    assert a.log_prob.shape == a.entropy.shape == (2, 3)
    assert a.top_log_prob.shape == a.top_index.shape == (2, 3, 2)
    assert torch.autograd.gradcheck(
        lambda v: ops.log_probs(v, t, top_k=2)[:3], z)
    one = ops.log_probs(z.detach()[0, 0], t[0, 0], top_k=1)
    assert one.log_prob.shape == () and one.top_index.shape == (1,)
    # the loss of a classifier
    ref = torch.nn.functional.cross_entropy(z.view(6, 5), t.view(6))
    assert torch.allclose(-a.log_prob.mean(), ref)


def test_log_probs_refusals():
    z = torch.zeros(3, 4)
    for args in ((z, torch.zeros(2, dtype=torch.int64)),
                 (z, torch.zeros(3)), (z.long(), None),
                 (z, torch.zeros(3, dtype=torch.bool)),
                 (z[:, :0], None)):
        with pytest.raises(AssertionError):
            ops.log_probs(*args)
    for k in (-1, 5):
        with pytest.raises(AssertionError):
            ops.log_probs(z, None, top_k=k)


@pytest.mark.parametrize("groups", [1, 5000, 16384])
def test_no_slots(groups):
    route = ops.route_rows(torch.empty(0, 2, dtype=torch.int64), groups)
    assert route.offsets.shape == (groups + 1,) and not route.offsets.any()
    assert route.position.shape == (0, 2) and route.source.shape == (0,)
    out = ops.combine_rows(route, ops.dispatch_rows(route, torch.zeros(0, 8)))
    assert out.shape == (0, 8)
