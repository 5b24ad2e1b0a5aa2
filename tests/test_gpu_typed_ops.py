"""The HIP kernels of the typed-row operators and of log_probs against plain
computations in 64 bits, at the sizes, strides and masks where they can go
wrong; on other streams and inside captured graphs."""
import math

import pytest
import torch

import typed_oracle as oracle
from test_typed_ops import ROWS, check_log_probs

from dgl_operator_amd import ops
from dgl_operator_amd.ops import backend

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    assert backend.has_extension(), "HIP extension must be built on GPU boxes"
    return torch.device("cuda:0")


def within(got, ref_tol):
    ref, tol = ref_tol
    got = got.detach().cpu().double()
    assert got.shape == ref.shape
    worst = ((got - ref).abs() - tol).max() if got.numel() else torch.tensor(0.)
    assert worst <= 0, f"off by {float(worst)} more than the bound"


def strided(t, how):
    """The same rows with another layout."""
    if how == "wide":      # a slice of wider rows, 16-byte aligned
        return torch.cat((t, t), 1)[:, :t.shape[1]]
    if how == "odd":       # rows that start one element off
        buf = t.new_zeros(t.shape[0], t.shape[1] + 1)
        buf[:, 1:] = t
        return buf[:, 1:]
    if how == "transposed":
        return t.t().contiguous().t()
    return t


# ---------------------------------------------------------------------------
# route
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows,k,groups", [
    (0, 2, 3), (1, 1, 1), (1, 2, 8), (63, 1, 5), (64, 3, 64), (1000, 2, 16),
    (4096, 2, 4096), (4096, 2, 1024), (8193, 1, 3), (20000, 2, 1345), (3000, 4, 16384),
    (40000, 1, 5000),
])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_route_rows(dev, rows, k, groups, dtype):
    ids = torch.randint(-1, groups + 1, (rows, k), dtype=dtype)
    got = ops.route_rows(ids.to(dev), groups)
    offsets, position, source = oracle.route(ids, groups)
    assert got.offsets.dtype == torch.int64
    assert torch.equal(got.offsets.cpu(), offsets)
    assert torch.equal(got.position.cpu(), position.view(rows, k))
    assert torch.equal(got.source.cpu(), source)


def test_route_rows_one_group_and_none(dev):
    """All slots in one group, and none in any; ids beyond 32 bits are none."""
    for n in (5000, 70000):
        for fill in (7, -1, 2 ** 32 + 7):
            ids = torch.full((n,), fill, device=dev)
            got = ops.route_rows(ids, 9)
            kept = n if fill == 7 else 0
            assert got.offsets.tolist() == [0] * 8 + [kept] * 2
            want = torch.arange(n, dtype=torch.int32)
            want = want if kept else torch.full_like(want, -1)
            assert torch.equal(got.position[:, 0].cpu(), want)
            assert torch.equal(got.source.cpu(), want)


def test_route_rows_refuses(dev):
    ids = torch.zeros(4, dtype=torch.int64, device=dev)
    with pytest.raises(RuntimeError, match="groups"):
        ops.route_rows(ids, 16385)
    route = ops.route_rows(ids, 2)
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        ops.dispatch_rows(route, torch.zeros(4, 2, device=dev).double())
    with pytest.raises(AssertionError):
        ops.dispatch_rows(route, torch.zeros(4, 2))
    with pytest.raises(AssertionError):
        ops.combine_rows(route, torch.zeros(4, 2, device=dev), torch.zeros(4))


def test_plans_made_by_hand_stay_inside(dev):
    """Positions that leave the sorted rows are dropped, never followed; other
    layouts than the plan's own are refused."""
    good = ops.route_rows(torch.tensor([[0, 1], [1, 0]], device=dev), 2)
    x, y = torch.ones(2, 8, device=dev), torch.ones(4, 8, device=dev)
    bad = good._replace(position=torch.tensor(
        [[4, 2 ** 31 - 1], [-7, 0]], dtype=torch.int32, device=dev))
    assert ops.dispatch_rows(bad, x).shape == (4, 8)
    assert torch.equal(ops.combine_rows(bad, y)[:, 0].cpu(),
                       torch.tensor([0.0, 1.0]))
    yr, w = y.clone().requires_grad_(), torch.ones(2, 2, device=dev)
    torch.autograd.grad(ops.combine_rows(bad, yr, w).sum(), yr)
    torch.cuda.synchronize()
    turned = good._replace(position=good.position.t())
    for call in (lambda: ops.dispatch_rows(turned, x),
                 lambda: ops.combine_rows(turned, y),
                 lambda: ops.combine_rows(
                     good._replace(position=good.position.long()), y)):
        with pytest.raises(RuntimeError, match="the plan's contiguous"):
            call()


@pytest.mark.parametrize("rows,k,width", [
    (1, 1, 1), (1, 2, 256), (5, 3, 7), (700, 2, 100), (513, 1, 47),
    (300, 4, 1030), (9, 2, 0), (0, 2, 16), (2000, 2, 64), (33, 20, 36),
])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", ["plain", "wide", "odd", "transposed"])
def test_dispatch_combine(dev, rows, k, width, dtype, how):
    ids = torch.randint(-1, 6, (rows, k))
    route = ops.route_rows(ids.to(dev), 5)
    position = route.position.cpu()
    x = torch.randn(rows, width).to(dtype)
    y = torch.randn(rows * k, width).to(dtype)
    w = torch.rand(rows, k)
    gs, go = torch.randn(rows * k, width).to(dtype), torch.randn(rows, width).to(dtype)
    xd, yd, gsd, god = (strided(t.to(dev), how) for t in (x, y, gs, go))
    wd = w.to(dev)
    for t in (xd, yd, wd):
        t.requires_grad_()
    xs = ops.dispatch_rows(route, xd)
    assert torch.equal(xs.detach().cpu(), oracle.dispatch(x, position))
    out = ops.combine_rows(route, yd, wd)
    within(out, oracle.combine(y, position, w))
    within(ops.combine_rows(route, yd), oracle.combine(y, position, None))
    dx, dy, dw = torch.autograd.grad((xs, out), (xd, yd, wd), (gsd, god))
    within(dx, oracle.combine(gs, position, None))
    ref = torch.zeros(rows * k, width, dtype=torch.float64)
    for f, p in enumerate(position.reshape(-1).tolist()):
        if p >= 0:
            ref[p] = w.reshape(-1)[f].double() * go[f // k].double()
    within(dy, (ref, (oracle.half(dtype) + 2 * oracle.U) * ref.abs()
                + oracle.tiny(dtype)))
    terms = oracle.taken(y, position) * go.double()[:, None, :]
    within(dw, (terms.sum(2), (width + 2) * oracle.U * terms.abs().sum(2)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_combine_weights_in_the_rows_type_and_alone(dev, dtype):
    """Weights of any float type; gradients of one input only."""
    ids = torch.randint(0, 4, (50, 2))
    route = ops.route_rows(ids.to(dev), 4)
    y = torch.randn(100, 24).to(dtype)
    w = torch.rand(50, 2).to(dtype)
    for need_y, need_w in ((True, False), (False, True)):
        yd, wd = y.to(dev).requires_grad_(need_y), w.to(dev).requires_grad_(need_w)
        out = ops.combine_rows(route, yd, wd)
        within(out, oracle.combine(y, route.position.cpu(), w))
        g, = torch.autograd.grad(out.float().sum(), yd if need_y else wd)
        assert g.dtype == dtype
        taken = oracle.taken(y, route.position.cpu())
        if need_w:
            s = taken.sum(2)
            within(g, (s, (26 * oracle.U + oracle.half(dtype))
                       * taken.abs().sum(2)))
        else:
            ref = torch.zeros(100, 24, dtype=torch.float64)
            ref[route.position.cpu().reshape(-1).long()] = \
                w.double().reshape(-1, 1).expand(100, 24)
            within(g, (ref, torch.zeros_like(ref)))


def test_rows_of_no_group_do_not_spread(dev):
    """NaN in rows that no slot takes reaches nothing."""
    ids = torch.tensor([[0, -1], [-1, -1], [1, 0]], device=dev)
    route = ops.route_rows(ids, 2)
    x = torch.ones(3, 8, device=dev)
    x[1] = math.nan
    xs = ops.dispatch_rows(route, x)
    assert torch.isfinite(xs).all() and not xs[3:].any()
    y = torch.full((6, 8), math.nan, device=dev)
    y[:3] = 1.0
    out = ops.combine_rows(route, y)
    assert torch.equal(out[:, 0].cpu(), torch.tensor([1.0, 0.0, 2.0]))


# ---------------------------------------------------------------------------
# segment_mm
# ---------------------------------------------------------------------------
def offsets_of(sizes, first=0):
    return torch.tensor([first] + list(sizes)).cumsum(0)


SHAPES = [
    # sizes, K, N, rows before, rows behind
    ([1], 1, 1, 0, 0),
    ([16], 256, 512, 0, 0),
    ([0, 0, 3], 7, 5, 1, 2),
    ([1, 2, 0, 5, 63, 64, 65, 1], 100, 47, 0, 0),
    ([2, 1, 2, 3, 2, 1, 3, 2], 256, 512, 0, 0),
    ([300, 0, 17], 33, 130, 5, 7),
    ([127, 129, 256, 1], 128, 128, 0, 0),
    ([1000, 24], 200, 264, 0, 3),
    ([700, 300, 24], 512, 136, 0, 0),
    ([40] * 30, 72, 40, 0, 0),
    ([5000], 16, 16, 0, 0),
    ([2100, 0, 520], 136, 264, 0, 2),
    ([1100], 264, 320, 1, 0),
    ([0, 700, 0, 3300, 1, 0], 256, 520, 40, 9),
]


@pytest.mark.parametrize("sizes,K,N,before,behind", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", ["plain", "odd", "weights transposed"])
def test_segment_mm(dev, sizes, K, N, before, behind, dtype, how):
    offsets = offsets_of(sizes, before)
    rows = int(offsets[-1]) + behind
    x, g = torch.randn(rows, K).to(dtype), torch.randn(rows, N).to(dtype)
    w = (torch.randn(len(sizes), K, N) * K ** -0.5).to(dtype)
    xd, gd, wd = x.to(dev), g.to(dev), w.to(dev)
    if how == "odd":
        xd, gd = strided(xd, "odd"), strided(gd, "odd")
        buf = torch.zeros(len(sizes), K, N + 1, dtype=dtype, device=dev)
        buf[:, :, 1:] = wd
        wd = buf[:, :, 1:]
    elif how == "weights transposed":
        wd = wd.transpose(1, 2).contiguous().transpose(1, 2)
    # what lies in rows of no group reaches nothing
    xd, gd = xd.clone() if how == "plain" else xd, gd
    if how == "plain":
        gd = gd.clone()
        for t in (xd, gd):
            t[:before] = math.nan
            t[rows - behind:] = math.nan
    xd.requires_grad_()
    wd.requires_grad_()
    y = ops.segment_mm(offsets.to(dev), xd, wd)
    within(y, oracle.segment_mm(offsets, x, w))
    dx, dw = torch.autograd.grad(y, (xd, wd), gd)
    within(dx, oracle.segment_mm(offsets, g, w.transpose(1, 2)))
    within(dw, oracle.segment_wgrad(offsets, x, g))


def test_segment_mm_nothing(dev):
    for rows, K, N in ((0, 4, 4), (3, 0, 4), (3, 4, 0)):
        offsets = torch.tensor([0, rows], device=dev)
        x = torch.randn(rows, K, device=dev, requires_grad=True)
        w = torch.randn(1, K, N, device=dev, requires_grad=True)
        y = ops.segment_mm(offsets, x, w)
        assert y.shape == (rows, N) and not y.any()
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert dx.shape == x.shape and dw.shape == w.shape and not dw.any()


def test_segment_mm_not_finite_stays_in_its_row(dev):
    """Partial tiles read nothing of their neighbours into their sums."""
    for dtype in TYPES:
        offsets = offsets_of([5, 70, 3])
        x = torch.randn(78, 40).to(dtype)
        x[4], x[5], x[77, 39] = math.nan, math.inf, math.nan
        w = torch.ones(3, 40, 24, dtype=dtype)
        y = ops.segment_mm(offsets.to(dev), x.to(dev), w.to(dev)).cpu()
        bad = ~torch.isfinite(y)
        assert bad[[4, 5, 77]].all()
        bad[[4, 5, 77]] = False
        assert not bad.any()


def test_segment_mm_bad_offsets_stay_inside(dev):
    """Offsets that leave the rows or fall are clamped, never followed."""
    x = torch.ones(10, 8, device=dev)
    w = torch.ones(2, 8, 8, device=dev)
    ok = ops.segment_mm(torch.tensor([-5, 4, 99], device=dev), x, w)
    assert torch.equal(ok, torch.full_like(ok, 8.0))
    for o in ([9, 3, 10], [4, 99, -1]):
        ops.segment_mm(torch.tensor(o, device=dev), x, w)
    torch.cuda.synchronize()


def test_segment_mm_refuses(dev):
    o = torch.tensor([0, 2], device=dev)
    x = torch.zeros(2, 3, device=dev)
    w = torch.zeros(1, 3, 4, device=dev)
    for bad in ((o.cpu(), x, w), (o, x.cpu(), w), (o, x, w.cpu())):
        with pytest.raises(AssertionError):
            ops.segment_mm(*bad)
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        ops.segment_mm(o, x.double(), w.double())


# ---------------------------------------------------------------------------
# log_probs
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("name", sorted(ROWS))
@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_rows(dev, name, dtype):
    z = torch.tensor([ROWS[name]] * 3)
    z = z.clamp(min=torch.finfo(dtype).min).where(z > -math.inf, z) \
        .clamp(max=torch.finfo(dtype).max).to(dtype)
    check_log_probs(dev, z, torch.tensor([0, 2, 4]), 5)


@pytest.mark.parametrize("rows,C", [
    (1, 1), (3, 2), (70, 47), (5, 64), (5, 65), (300, 100), (6, 129),
    (4, 512), (3, 1000), (3, 1345), (2, 4097), (2, 14951), (1, 16385),
    (2, 40001),
])
@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_sizes(dev, rows, C, dtype):
    z = torch.randn(rows, C) * 3
    if C > 2:
        hide = torch.rand(rows, C) < 0.2
        hide[:, C // 2] = False
        z.masked_fill_(hide, -math.inf)
    z = z.to(dtype)
    t = torch.randint(0, C, (rows,))
    for k in {0, 1, min(C, 5), min(C, 10), min(C, 15), min(C, 20), min(C, 32)}:
        check_log_probs(dev, z, t, k)
    check_log_probs(dev, z, None, min(C, 3))


@pytest.mark.parametrize("C", [47, 300, 3000, 20000])
@pytest.mark.parametrize("pattern", ["equal", "rising", "falling", "few"])
def test_log_probs_ties_and_orders(dev, C, pattern):
    """Rows whose best classes are many, first, last or equal."""
    j = torch.arange(C, dtype=torch.float32)
    z = {"equal": torch.zeros(C), "rising": j / C, "falling": -j / C,
         "few": (j % 3)}[pattern][None].repeat(2, 1)
    check_log_probs(dev, z, torch.tensor([0, C - 1]), 32)


@pytest.mark.parametrize("C", [6, 200, 5000, 20000])
def test_log_probs_targets(dev, C):
    z = torch.randn(6, C)
    t = torch.tensor([1, -100, C, -1, 2 ** 40, -(2 ** 63)])
    check_log_probs(dev, z, t, 2)
    check_log_probs(dev, z, torch.tensor([1, 5, 5, 0, 2, 5]), 0, ignore=5)


@pytest.mark.parametrize("C", [3, 120, 700, 5000, 20000])
@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_not_finite(dev, C, dtype):
    z = torch.randn(4, C).to(dtype)
    z[0, 1] = math.nan
    z[1, C - 1] = math.inf
    z[3] = -math.inf
    z[3, 2] = math.nan
    zd = z.to(dev).requires_grad_()
    a = ops.log_probs(zd, torch.zeros(4, dtype=torch.int64, device=dev), top_k=2)
    bad = [True, True, False, True]
    for o in (a.log_prob, a.entropy, a.top_log_prob[:, 0]):
        assert o.isnan().tolist() == bad
    _, _, _, index, _ = oracle.log_probs(z, None, 2)
    assert torch.equal(a.top_index.cpu(), index)
    g, = torch.autograd.grad(a.log_prob.sum(), zd)
    assert g.isnan().all(1).tolist() == bad


@pytest.mark.parametrize("how", ["wide", "odd", "transposed", "one row"])
@pytest.mark.parametrize("C", [47, 1000, 14951])
def test_log_probs_strides(dev, how, C):
    z = torch.randn(5, C)
    if how == "one row":
        zd = z[:1].to(dev).expand(5, C)
        z = z[:1].expand(5, C)
    else:
        zd = strided(z.to(dev), how)
    t = torch.randint(0, C, (5,))
    a = ops.log_probs(zd, t.to(dev), top_k=3)
    b = ops.log_probs(z.contiguous().to(dev), t.to(dev), top_k=3)
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    zd = zd.detach().requires_grad_()
    a = ops.log_probs(zd, t.to(dev), top_k=3)
    g, = torch.autograd.grad(a.log_prob.sum() + a.entropy.sum(), zd)
    assert g.shape == zd.shape and torch.isfinite(g).all()


def test_log_probs_partial_gradients(dev):
    """Each output alone, and gradients that are broadcast."""
    z = torch.randn(9, 50, device=dev, requires_grad=True)
    t = torch.randint(0, 50, (9,), device=dev)
    zc = z.detach().cpu().double().requires_grad_()
    for i in range(3):
        a = ops.log_probs(z, t, top_k=4)
        b = ops.log_probs(zc, t.cpu(), top_k=4)
        g, = torch.autograd.grad(a[i].sum(), z)
        h, = torch.autograd.grad(b[i].sum(), zc)
        # p and log p within 64 roundings of at most ~10, sums of 4
        assert (g.cpu().double() - h).abs().max() < 64 * 10 * 4 * oracle.U


def test_log_probs_strided_targets(dev):
    z = torch.randn(5, 3, 7, device=dev)
    t = torch.randint(0, 7, (3, 5), device=dev)
    a = ops.log_probs(z, t.t())
    b = ops.log_probs(z.reshape(15, 7), t.t().reshape(15).int())
    assert torch.equal(a.log_prob.reshape(15), b.log_prob)
    c = ops.log_probs(z[:, 0], t[0].repeat_interleave(2)[::2])
    assert torch.equal(c.log_prob, a.log_prob[:, 0])


def test_second_derivatives_are_refused(dev):
    """A first derivative may be part of a graph; a second one raises."""
    x = torch.randn(4, 6, device=dev, requires_grad=True)
    w = torch.randn(2, 6, 6, device=dev, requires_grad=True)
    p = torch.rand(4, 1, device=dev, requires_grad=True)
    route = ops.route_rows(torch.tensor([0, 1, 1, 0], device=dev), 2)
    for y in (ops.dispatch_rows(route, x), ops.combine_rows(route, x, p),
              ops.segment_mm(route.offsets, x, w),
              ops.log_probs(x).entropy):
        g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            g.sum().backward()


def test_log_probs_refuses(dev):
    z = torch.zeros(3, 40, device=dev)
    with pytest.raises(RuntimeError, match="top_k"):
        ops.log_probs(z, None, top_k=33)
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        ops.log_probs(z.double())
    with pytest.raises(AssertionError):
        ops.log_probs(z, torch.zeros(3, dtype=torch.int64))


# ---------------------------------------------------------------------------
# offsets beyond 32 bits, streams, graphs, the operators together
# ---------------------------------------------------------------------------
def test_rows_beyond_32_bits(dev):
    """Rows whose elements lie past 2^31: the last rows of wide strides."""
    rows, stride = 600_000, 4096
    big = torch.zeros(rows, stride, dtype=torch.bfloat16, device=dev)
    x = big[:, :16]
    x[-70:] = torch.randn(70, 16, device=dev).to(torch.bfloat16)
    last = x[-70:].cpu()
    ids = torch.full((rows,), -1, device=dev)
    ids[-70:] = torch.arange(70, device=dev) % 3
    route = ops.route_rows(ids, 3)
    xs = ops.dispatch_rows(route, x)
    order = torch.cat([torch.arange(g, 70, 3) for g in range(3)])
    assert torch.equal(xs[:70].cpu(), last[order]) and not xs[70:].any()
    offsets = torch.tensor([rows - 70, rows - 3, rows], device=dev)
    w = torch.randn(2, 16, 8, dtype=torch.bfloat16)
    y = ops.segment_mm(offsets, x, w.to(dev))
    assert not y[:-70].any()
    within(y[-70:], oracle.segment_mm(torch.tensor([0, 67, 70]), last, w))
    dw = ops.segment_mm.__globals__["backend"].load_extension().segment_mm_wgrad(
        offsets, x, y)
    within(dw, oracle.segment_wgrad(torch.tensor([0, 67, 70]), last, y[-70:].cpu()))
    a = ops.log_probs(x, torch.full((rows,), 3, device=dev), top_k=2)
    lp, _, _, index, _ = oracle.log_probs(last, torch.full((70,), 3), 2)
    assert torch.equal(a.top_index[-70:].cpu(), index)
    assert (a.log_prob[-70:].cpu().double() - lp).abs().max() < 400 * oracle.U


def mixture(ids_from, x, router, w1, w2, target, groups, k):
    """A top-k mixture of experts and its loss, by the operators."""
    whole = torch.arange(2, device=x.device) * x.shape[0]
    gate = ops.log_probs(ops.segment_mm(whole, x, router[None]), None, top_k=k)
    route = ops.route_rows(gate.top_index if ids_from is None else ids_from,
                           groups)
    xs = ops.dispatch_rows(route, x)
    h = torch.tanh(ops.segment_mm(route.offsets, xs, w1))
    ys = ops.segment_mm(route.offsets, h, w2)
    out = ops.combine_rows(route, ys, gate.top_log_prob.exp())
    answer = ops.log_probs(out, target)
    return out, answer.log_prob.mean() + 0.01 * gate.entropy.mean()


def mixture_plain(x, router, w1, w2, target, k):
    p = torch.softmax(x @ router, 1)
    index = torch.sort(p, dim=1, descending=True, stable=True).indices[:, :k]
    all_out = torch.tanh(torch.einsum("td,gdh->tgh", x, w1))
    all_out = torch.einsum("tgh,gho->tgo", all_out, w2)
    rows = torch.arange(x.shape[0])[:, None]
    out = (all_out[rows, index] * p[rows, index][:, :, None]).sum(1)
    lp = torch.log_softmax(out, 1)[torch.arange(x.shape[0]), target]
    entropy = -(p * p.log()).sum(1)
    return out, lp.mean() + 0.01 * entropy.mean()


def mixture_inputs(rows, groups=6, d=40, h=24, o=47):
    gen = torch.Generator().manual_seed(3)
    make = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return (make(rows, d), make(d, groups) / 6, make(groups, d, h) / 6,
            make(groups, h, o) / 5,
            torch.randint(0, o, (rows,), generator=gen))


@pytest.mark.parametrize("rows", [1, 33, 700])
def test_mixture_of_experts_together(dev, rows):
    """Router, dispatch, experts, combine and loss against 64 bits."""
    ins = mixture_inputs(rows)
    gpu = [t.to(dev).requires_grad_(t.is_floating_point()) for t in ins]
    wide = [t.double().requires_grad_() if t.is_floating_point() else t
            for t in ins]
    out, loss = mixture(None, *gpu, 6, 2)
    ref, ref_loss = mixture_plain(*wide, 2)
    got = torch.autograd.grad(loss, gpu[:4])
    want = torch.autograd.grad(ref_loss, wide[:4])
    # sums of 40 and 24 products whose terms add up to at most ~4 times the
    # largest result: (42 + 26) * 4 U for the experts, 42 * 4 U in the router's
    # logits and so in the weights; the way back doubles each: < 1600 U
    for a, b in zip((out, loss, *got), (ref, ref_loss, *want)):
        assert (a.detach().cpu().double() - b).abs().max() <= \
            1600 * oracle.U * b.abs().max()


def test_mixture_on_another_stream(dev):
    ins = [t.to(dev) for t in mixture_inputs(300)]
    want, _ = mixture(None, *ins, 6, 2)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [mixture(None, *ins, 6, 2)[0] for _ in range(3)]
    s.synchronize()
    for g in got:
        assert torch.equal(g, want)


def test_mixture_on_two_streams_at_once(dev):
    """Two programs side by side share nothing."""
    ins = [[t.to(dev) for t in mixture_inputs(n)] for n in (400, 900)]
    want = [mixture(None, *i, 6, 2)[0] for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = [[], []]
    for _ in range(5):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(mixture(None, *ins[n], 6, 2)[0])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for t in g:
            assert torch.equal(t, w)


def test_gradients_of_one_side_and_shared_weights(dev):
    """Each input's gradient alone; one weight expanded over all groups, whose
    gradient is the sum over them; an output's gradient that is a broadcast."""
    offsets = offsets_of([700, 1, 0, 340]).to(dev)
    x = torch.randn(1041, 136, device=dev).bfloat16()
    w = (torch.randn(136, 264, device=dev) / 12).bfloat16()
    for need_x, need_w in ((True, False), (False, True)):
        xd = x.clone().requires_grad_(need_x)
        wd = w.clone().requires_grad_(need_w)
        y = ops.segment_mm(offsets, xd, wd.expand(4, 136, 264))
        within(y, oracle.matmul(x.cpu(), w.cpu(), x.dtype))
        g, = torch.autograd.grad(y, xd if need_x else wd,
                                 torch.ones(1, 1, device=dev).bfloat16()
                                 .expand(1041, 264))
        ones = torch.ones(1041, 264).bfloat16()
        if need_x:
            within(g, oracle.matmul(ones, w.cpu().t(), x.dtype))
        else:
            ref, tol = oracle.matmul(x.cpu().t(), ones, x.dtype)
            # four groups' gradients, each rounded, and their sum rounded
            # thrice: at most 4 + 3 halves of a step of sums of |x|
            size = x.cpu().double().abs().sum(0)[:, None]
            within(g, (ref, tol + 7 * oracle.half(x.dtype) * size))


def test_mixture_captured(dev):
    """One graph with forward and backward, replayed with new inputs between
    eager runs of the same program; another graph shares nothing with it."""
    ins = [t.to(dev) for t in mixture_inputs(200)]

    def step(ts):
        leaves = [t.detach().requires_grad_() for t in ts[:4]]
        out, loss = mixture(None, *leaves, ts[4], 6, 2)
        return (out, loss) + torch.autograd.grad(loss, leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(ins)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(ins)
        graphs.append((graph, outs))
    for i in range(4):
        ins[0].copy_(torch.randn(ins[0].shape, device=dev))
        want = step([t.clone() for t in ins])
        torch.cuda.synchronize()
        for graph, outs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_runs_repeat_bit_for_bit(dev):
    ins = [t.to(dev) for t in mixture_inputs(5000)]
    runs = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in ins[:4]]
        out, loss = mixture(None, *leaves, ins[4], 6, 2)
        runs.append((out,) + torch.autograd.grad(loss, leaves[2:]))
    for r in runs[1:]:
        for a, b in zip(r, runs[0]):
            assert torch.equal(a, b)
