"""Calls at the edges of the typed-row operators and of log_probs on the GPU:
finite masks that fill a part of a long row, large gradients, empty batches,
launches of more threads than one grid holds, gradients that nobody asked for."""
import math

import pytest
import torch

import typed_oracle as oracle
from test_gpu_typed_variants import check_mm
from test_typed_ops import check_log_probs

from dgl_operator_amd import ops
from dgl_operator_amd.ops import backend

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    assert backend.has_extension(), "HIP extension must be built on GPU boxes"
    return torch.device("cuda:0")


@pytest.mark.parametrize("C", [16400, 20000, 40001])
@pytest.mark.parametrize("dtype", TYPES)
def test_parts_of_a_long_row_far_apart(dev, C, dtype):
    """Parts of a split row whose values lie as far apart as the type lets them:
    a range of classes masked by the lowest value, at either end or in the
    middle, a row that is lowest but for one, one that is highest but for one."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    z = torch.randn(6, C)
    z[0, C // 2 - 16:] = low
    z[1, :C // 2 + 16] = low
    z[2, C // 3:C - C // 3] = low
    z[3] = low
    z[3, C - 1] = 1.0
    z[4] = high
    z[4, 0] = low
    z[5, :C - 8] = -math.inf
    z = z.to(dtype)
    t = torch.tensor([3, C - 2, 1, C - 1, 7, C - 3])
    for k in (0, 5):
        check_log_probs(dev, z, t, k)


@pytest.mark.parametrize("C", [20, 300, 5000, 20000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_entropy_gradients(dev, C, dtype):
    """A scaled loss: the gradient is linear in the entropy's, so that a power
    of two goes through it exactly, also where a class was taken away."""
    z = torch.randn(5, C)
    z[:, ::3] = -math.inf
    z[1] = torch.finfo(dtype).min
    z[1, 4] = 0.0
    z[2] = -math.inf
    zd = z.to(dtype).to(dev).requires_grad_()
    ent = ops.log_probs(zd).entropy
    small, = torch.autograd.grad(ent, zd, torch.ones_like(ent),
                                 retain_graph=True)
    large, = torch.autograd.grad(ent, zd, torch.full_like(ent, 2.0 ** 33))
    assert torch.isfinite(large).all()
    assert torch.equal(large, small * 2.0 ** 33)


def peak_of(call):
    """Bytes that a call holds at most beyond what was there."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


def test_gradients_that_nobody_asks_for(dev):
    """Both inputs may learn; a backward pass makes the gradients asked for and
    does not hold the others'."""
    offsets = torch.tensor([0, 100, 400], device=dev)
    x = torch.randn(400, 512, device=dev, requires_grad=True)
    w = torch.randn(2, 512, 4096, device=dev, requires_grad=True)
    y = ops.segment_mm(offsets, x, w)
    g = torch.ones_like(y)
    (dx,), held = peak_of(lambda: torch.autograd.grad(y, x, g, retain_graph=True))
    assert held < 2 * x.numel() * 4, "dw is 16 times dx"
    both = torch.autograd.grad(y, (x, w), g, retain_graph=True)
    assert torch.equal(dx, both[0])
    (dw,), _ = peak_of(lambda: torch.autograd.grad(y, w, g))
    assert torch.equal(dw, both[1])

    ids = torch.randint(0, 4, (3000, 2), device=dev)
    route = ops.route_rows(ids, 4)
    rows = torch.randn(6000, 256, device=dev, requires_grad=True)
    weights = torch.rand(3000, 2, device=dev, requires_grad=True)
    out = ops.combine_rows(route, rows, weights)
    g = torch.randn_like(out)
    (dweights,), held = peak_of(
        lambda: torch.autograd.grad(out, weights, g, retain_graph=True))
    assert held < rows.numel() * 4 // 2
    (drows,), _ = peak_of(
        lambda: torch.autograd.grad(out, rows, g, retain_graph=True))
    both = torch.autograd.grad(out, (rows, weights), g)
    assert torch.equal(drows, both[0]) and torch.equal(dweights, both[1])


@pytest.mark.parametrize("groups", [1, 3, 4096, 4097, 5000, 16384])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_no_slots(dev, groups, dtype):
    """An empty batch, however many groups there are, and the operators on it."""
    for k in (1, 2):
        ids = torch.empty(0, k, dtype=dtype, device=dev)
        # the block that the offsets take next is not zero by chance
        del_me = torch.full((groups + 1,), 7, device=dev)
        del del_me
        route = ops.route_rows(ids, groups)
        assert route.offsets.shape == (groups + 1,) and not route.offsets.any()
        assert route.position.shape == (0, k) and route.source.shape == (0,)
        x = torch.zeros(0, 8, device=dev, requires_grad=True)
        w = torch.ones(groups, 8, 4, device=dev, requires_grad=True)
        y = ops.segment_mm(route.offsets, ops.dispatch_rows(route, x), w)
        out = ops.combine_rows(route, y)
        assert out.shape == (0, 4)
        dx, dw = torch.autograd.grad(out.sum(), (x, w))
        assert dx.shape == (0, 8) and not dw.any()


def sliding(dev, rows, C, dtype=torch.bfloat16):
    """rows x C logits, each row one element further on: no memory to speak of."""
    line = torch.randn(rows + C, device=dev).to(dtype)
    return line.as_strided((rows, C), (1, 1))


def check_windows(z, t, k, marks, g=None):
    """Rows around the marks are what a call of those rows alone gives."""
    zr = z.detach().requires_grad_(g is not None)
    a = ops.log_probs(zr, t, top_k=k)
    dz = None
    if g is not None:
        dz, = torch.autograd.grad((a.log_prob, a.entropy), zr, g)
    for m in marks:
        at = slice(max(0, m - 20), min(z.shape[0], m + 20))
        part = z[at].contiguous().requires_grad_(g is not None)
        b = ops.log_probs(part, t[at], top_k=k)
        for u, v in zip(a, b):
            assert torch.equal(u[at], v), f"row {m}"
        if g is not None:
            d, = torch.autograd.grad((b.log_prob, b.entropy), part,
                                     [v[at] for v in g])
            assert torch.equal(dz[at], d), f"gradient of row {m}"


@pytest.mark.parametrize("rows,C,k", [(2_150_000, 20000, 3),
                                      (268_440_000, 257, 1)])
def test_more_threads_than_one_grid(dev, rows, C, k):
    """2^32 threads and more: a block of 1024 a part of a long row, sixteen lanes
    a short one."""
    lanes = 2 * 1024 if C == 20000 else 16
    edge = (2 ** 32 - 1024) // lanes
    assert rows > edge
    z = sliding(dev, rows, C)
    t = torch.randint(0, C, (rows,), device=dev)
    check_windows(z, t, k, [0, rows // 3, edge - 10, edge, edge + 10, rows])
    torch.cuda.empty_cache()


def test_more_threads_than_one_grid_backward(dev):
    """Two gradient tiles of 256 threads a row (and one block of 1024 forward)."""
    rows, C = 8_390_000, 4097
    back, front = (2 ** 32 - 1024) // 512, (2 ** 32 - 1024) // 1024
    assert rows > back > front
    z = sliding(dev, rows, C)
    t = torch.randint(0, C, (rows,), device=dev)
    g = [torch.randn(rows, device=dev) for _ in range(2)]
    check_windows(z, t, 0, [0, front, back, rows // 3, rows], g)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
def test_more_groups_than_a_grid_is_high(dev, dtype):
    """70000 groups of a row or so, and none in some."""
    G, K, N = 70_000, 8, 12
    gen = torch.Generator().manual_seed(1)
    sizes = torch.randint(0, 3, (G,), generator=gen)
    offsets = torch.cat((torch.zeros(1).long(), sizes.cumsum(0))).to(dev)
    rows = int(offsets[-1])
    group = torch.repeat_interleave(torch.arange(G), sizes).to(dev)
    x = torch.randn(rows, K, device=dev).to(dtype).requires_grad_()
    w = torch.randn(G, K, N, device=dev).to(dtype).requires_grad_()
    g = torch.randn(rows, N, device=dev).to(dtype)
    y = ops.segment_mm(offsets, x, w)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    xw, gw, ww = x.detach().double(), g.double(), w.detach().double()[group]

    def close(got, terms, steps):
        ref, size = terms.sum(-1), terms.abs().sum(-1)
        acc = 2 * (steps + 2) * oracle.U * size
        tol = acc + oracle.half(dtype) * (ref.abs() + acc) + oracle.tiny(dtype)
        assert ((got.detach().double() - ref).abs() <= tol).all()

    close(y, xw[:, None, :] * ww.transpose(1, 2), K)
    close(dx, gw[:, None, :] * ww, N)
    outer = xw[:, :, None] * gw[:, None, :]
    ref = torch.zeros(G, K, N, dtype=torch.float64, device=dev)
    size = ref.index_add(0, group, outer.abs())
    ref.index_add_(0, group, outer)
    tol = 8 * oracle.U * size + oracle.half(dtype) * ref.abs() * 1.01 \
        + oracle.tiny(dtype)
    assert ((dw.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype,K,N", [(torch.float32, 16, 16),
                                       (torch.bfloat16, 128, 136)])
def test_many_groups_by_teams(dev, dtype, K, N):
    """More groups than the teams' sums have rows of blocks."""
    G = 1100
    mean = 256 if dtype == torch.float32 else 512
    sizes = [0 if e % 9 == 0 else mean + mean * (e % 5) // 4 for e in range(G)]
    assert sum(sizes) >= mean * G
    check_mm(dev, sizes, K, N, 0, 0, dtype, "plain")


def test_more_tiles_than_one_launch_holds(dev):
    """Refused before anything is allocated or launched."""
    rows = 2 ** 30 - 1
    x = torch.ones(1, 1, device=dev).expand(rows, 1)
    w = torch.ones(1, 1, 65, device=dev)
    offsets = torch.tensor([0, rows], device=dev)
    with pytest.raises(RuntimeError, match="too many tiles"):
        ops.segment_mm(offsets, x, w)
    G = 4_200_000
    w = torch.ones(1, 65, 65, device=dev).expand(G, 65, 65).requires_grad_()
    offsets = torch.ones(G + 1, dtype=torch.int64, device=dev)
    offsets[0] = 0
    y = ops.segment_mm(offsets, torch.ones(1, 65, device=dev), w)
    assert torch.equal(y, torch.full_like(y, 65.0))
    with pytest.raises(RuntimeError, match="too many tiles"):
        torch.autograd.grad(y.sum(), w)


def test_rows_too_wide_are_refused(dev):
    """Columns are counted in 32 bits: wider rows raise, nothing is left out."""
    route = ops.route_rows(torch.zeros(1, dtype=torch.int64, device=dev), 1)
    for width in (2 ** 30, 2 ** 31, 2 ** 32 + 8):
        x = torch.ones(1, 1, dtype=torch.bfloat16, device=dev).expand(1, width)
        with pytest.raises(RuntimeError, match="fewer than 2\\^30"):
            ops.dispatch_rows(route, x)
        with pytest.raises(RuntimeError, match="fewer than 2\\^30"):
            ops.combine_rows(route, x)
    x = torch.arange(2 ** 30 - 4, dtype=torch.int32, device=dev).to(torch.bfloat16)
    out = ops.combine_rows(route, ops.dispatch_rows(route, x[None]))
    assert torch.equal(out[0], x)
    del x, out
    torch.cuda.empty_cache()
