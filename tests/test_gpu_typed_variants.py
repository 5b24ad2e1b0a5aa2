"""Every variant that the sizes choose of segment_mm and log_probs, compared with
64-bit computations on the device. Each case states the rule that sends it to its
kernel, so that a changed rule shows here."""
import math

import pytest
import torch

import typed_oracle as oracle
from test_gpu_typed_ops import TYPES, offsets_of, strided

from dgl_operator_amd import ops
from dgl_operator_amd.ops import backend

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    assert backend.has_extension(), "HIP extension must be built on GPU boxes"
    return torch.device("cuda:0")


def cus():
    """Blocks of a kernel that fills the chip once."""
    return torch.cuda.get_device_properties(0).multi_processor_count // 8 * 8


def up(a, b):
    return -(-a // b)


def near(got, ref, tol, what=""):
    got = got.detach().double()
    assert got.shape == ref.shape
    same = (got == ref) | (got.isnan() & ref.isnan())
    bad = ~(same | ((got - ref).abs() <= tol))
    assert not bad.any(), \
        f"{what}: {int(bad.sum())} off, by {float((got - ref).abs()[bad].max())}"


# ---------------------------------------------------------------------------
# segment_mm
# ---------------------------------------------------------------------------
def product(a, b, dtype):
    """a @ b in 64 bits and the bound of its sums in fp32 (one rounding)."""
    a, b = a.double().contiguous(), b.double().contiguous()
    ref, size = a.mm(b), a.abs().mm(b.abs())
    acc = 2 * (a.shape[1] + 2) * oracle.U * size
    return ref, acc + oracle.half(dtype) * (ref.abs() + acc) + oracle.tiny(dtype)


def check_mm(dev, sizes, K, N, before, behind, dtype, how, backward=True):
    offsets = offsets_of(sizes, before)
    rows, G = int(offsets[-1]) + behind, len(sizes)
    gen = torch.Generator(device=dev).manual_seed(K * 7 + N)

    def make(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    x, g = make(rows, K).to(dtype), make(rows, N).to(dtype)
    w = (make(G, K, N) * K ** -0.5).to(dtype)
    # rows of no group hold what must reach nothing
    for t in (x, g):
        t[:before] = math.nan
        t[rows - behind:] = math.nan
    xd, gd, wd = x, g, w
    if how in ("wide", "odd"):
        xd, gd = strided(x, how), strided(g, how)
        assert xd.stride(0) > K and gd.stride(0) > N
    if how == "turned":
        wd = w.transpose(1, 2).contiguous().transpose(1, 2)
    xd, wd = xd.detach().requires_grad_(), wd.detach().requires_grad_()
    y = ops.segment_mm(offsets.to(dev), xd, wd)
    ends = list(zip(offsets[:-1].tolist(), offsets[1:].tolist()))
    held = slice(before, rows - behind)
    assert not y[:before].any() and not y[rows - behind:].any()
    for e, (a, b) in enumerate(ends):
        near(y[a:b], *product(x[a:b], w[e], dtype), f"y of group {e}")
    if not backward:
        return
    dx, dw = torch.autograd.grad(y, (xd, wd), gd)
    assert torch.isfinite(dx[held]).all()
    assert not dx[:before].any() and not dx[rows - behind:].any()
    for e, (a, b) in enumerate(ends):
        near(dx[a:b], *product(g[a:b], w[e].t(), dtype), f"dx of group {e}")
        near(dw[e], *product(x[a:b].t(), g[a:b], dtype), f"dw of group {e}")


def uneven(groups, mean, seed=0):
    """Sizes between none and three times the mean, some of them none or one."""
    gen = torch.Generator().manual_seed(seed)
    sizes = (torch.rand(groups, generator=gen) ** 2 * 3 * mean).long()
    sizes[::7] = 0
    sizes[3::11] = 1
    return sizes.tolist()


@pytest.mark.parametrize("K,N", [(24, 4096), (40, 8200), (520, 4104)])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("how", ["plain", "turned", "wide"])
def test_long_groups_many_tiles(dev, K, N, dtype, how):
    """256 x 256 tiles, several a block: the ring runs on into the next tile,
    over tiles without rows and behind results on their way out."""
    sizes, before, behind = [1500, 0, 37, 1800, 0, 1, 900], 3, 5
    rows, tn = sum(sizes) + before + behind, up(N, 256)
    assert N >= 256 and rows >= 512 * len(sizes)
    blocks = cus() // 8
    full = sum(up(s, 256) for s in sizes) * tn
    assert full > 8 * blocks, "some block has a second tile"
    check_mm(dev, sizes, K, N, before, behind, dtype, how,
             backward=K >= 256 and how != "wide")


@pytest.mark.parametrize("sizes,K,N", [
    # 4 teams of 1056 rows: groups begin, end and lie whole inside them
    ([1500, 0, 37, 1800, 1, 862], 2048, 2048),
    # 4 teams, one group
    ([4200], 2048, 2040),
    # 128 teams, tiles that both widths leave
    (None, 136, 264),
])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("how", ["plain", "wide"])
def test_weight_gradient_of_long_groups(dev, sizes, K, N, dtype, how):
    """256 x 256 tiles of dW by teams of blocks, with planes."""
    sizes = uneven(160, 1300) if sizes is None else sizes
    before, behind = 3, 5
    rows = sum(sizes) + before + behind
    tiles = up(K, 256) * up(N, 256)
    assert K >= 128 and N >= 128 and rows >= 512 * len(sizes)
    assert tiles <= cus() and rows // (cus() // tiles) >= 1024
    assert cus() // tiles > 1
    check_mm(dev, sizes, K, N, before, behind, dtype, how)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", ["plain", "turned", "wide", "odd"])
def test_groups_of_about_seventy_rows(dev, dtype, how):
    """Tiles of 64 x 128 (16-bit) and 64 x 64 (fp32)."""
    sizes = [70, 65, 0, 1, 190, 64, 63, 100, 48, 129, 20, 128]
    rows = sum(sizes) + 3
    assert 48 * len(sizes) < rows <= 96 * len(sizes)
    for K, N in ((72, 136), (128, 256), (100, 47), (200, 400)):
        check_mm(dev, sizes, K, N, 1, 2, dtype, how)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", ["plain", "wide", "odd"])
def test_weight_gradient_tile_by_tile(dev, dtype, how):
    """dW by one block for each group and tile, in long steps: groups of more
    than 256 rows whose tiles fill the chip by themselves."""
    for sizes, K, N in (([300], 2944, 2944),
                        (uneven(150, 420), 584, 760)):
        rows, G = sum(sizes) + 3, len(sizes)
        assert 256 * G < rows < 512 * G
        side = 128 if dtype != torch.float32 and how != "odd" else 64
        blocks = (4 if side == 64 else 2) * cus()
        tiles = up(K, side) * up(N, side)
        assert up(blocks, tiles) <= 1 or tiles * G >= 8 * blocks
        check_mm(dev, sizes, K, N, 1, 2, dtype, how)


@pytest.mark.parametrize("dtype", TYPES)
def test_aligned_rows_of_a_wider_matrix(dev, dtype):
    """Chunks straight to LDS from rows whose stride is not their width."""
    for sizes, K, N in (([1, 2, 0, 5, 63, 64, 65, 1], 96, 48),
                        ([127, 129, 256, 1], 128, 128),
                        ([1000, 24], 200, 264), ([40] * 30, 72, 40),
                        ([5000], 16, 16), ([2100, 0, 520], 136, 264)):
        check_mm(dev, sizes, K, N, 2, 1, dtype, "wide")


# ---------------------------------------------------------------------------
# log_probs
# ---------------------------------------------------------------------------
def check_answers(dev, z, target, k, ignore=-100):
    """All rows, forward and backward, against 64 bits; the bounds are those of
    check_log_probs in test_typed_ops.py."""
    rows, C = z.shape
    u, s_err = oracle.U, oracle.log_s_error(z)
    zr = z.detach().requires_grad_()
    got = ops.log_probs(zr, target, top_k=k, ignore_index=ignore)
    wide = z.detach().double()
    none = (wide == -math.inf).all(1)
    logp = torch.where(none[:, None], wide, torch.log_softmax(wide, 1))
    p = logp.exp()
    ent = torch.where(none, 0.0, -torch.xlogy(p, p).sum(1))
    index = torch.sort(wide, dim=1, descending=True,
                       stable=True).indices[:, :k]
    inside = (target >= 0) & (target < C)
    at = target.clamp(0, C - 1)[:, None]
    lp = torch.where(inside, logp.gather(1, at)[:, 0], math.nan)
    lp = torch.where(target == ignore, 0.0, lp)
    assert torch.equal(got.top_index, index)
    spread = wide.amax(1, keepdim=True) - wide
    spread = torch.where(torch.isfinite(spread), spread, 0.0)
    tol = u * (2 * logp.abs() + spread) + s_err
    tol = torch.where(torch.isfinite(tol), tol, 0.0)
    near(got.log_prob, lp, tol.gather(1, at)[:, 0], "log_prob")
    near(got.top_log_prob, logp.gather(1, index), tol.gather(1, index), "top")
    mean = (p * spread).sum(1)
    ent_tol = 2 * s_err * (mean + 1) + 4 * u * (p * spread * spread).sum(1) \
        + 2 * u * (ent.abs() + mean)
    near(got.entropy, ent, ent_tol, "entropy")

    gen = torch.Generator(device=dev).manual_seed(rows + C)
    g = [torch.randn(rows, *tail, generator=gen, device=dev)
         for tail in ((), (), (k,))]
    (dz,) = torch.autograd.grad(got[:3], zr, g)
    assert dz.dtype == z.dtype and dz.shape == z.shape
    g = [v.double() for v in g]
    g_lp = torch.where(inside, g[0], math.nan)
    g_lp = torch.where(target == ignore, 0.0, g_lp)
    own = torch.zeros_like(wide).scatter_add_(
        1, at, torch.where(inside, g_lp, 0.0)[:, None])
    size = torch.zeros_like(wide).scatter_add_(
        1, at, torch.where(inside, g_lp, 0.0).abs()[:, None])
    own.scatter_add_(1, index, g[2])
    size.scatter_add_(1, index, g[2].abs())
    ref = own - p * (g_lp + g[2].sum(1))[:, None] - g[1][:, None] * (
        torch.xlogy(p, p) + p * ent[:, None])
    ref = torch.where(none[:, None], 0.0, ref)
    pulls = (g_lp.abs() + g[2].abs().sum(1)).nan_to_num(0.0)[:, None]
    fl = logp.abs() + ent.abs()[:, None]
    fl = torch.where(torch.isfinite(fl), fl, 0.0)
    rel = tol + 8 * u
    gtol = p * (pulls * (2 * rel + (k + 4) * u) + g[1].abs()[:, None]
                * (fl * (2 * rel + 8 * u) + tol + ent_tol[:, None]))
    gtol = gtol + (k + 4) * u * size
    gtol = torch.where(torch.isfinite(gtol), gtol, 0.0)
    near(dz, ref, gtol + oracle.half(z.dtype) * (ref.abs() + gtol)
         + oracle.tiny(z.dtype), "gradient")


def answers_of(dev, rows, C, dtype, how):
    """Logits with filtered classes, ties, a row without classes and one with a
    single one; targets of which some are ignored or outside."""
    gen = torch.Generator(device=dev).manual_seed(rows * 31 + C)
    z = torch.randn(rows, C, generator=gen, device=dev) * 3
    z[rows // 2:rows // 2 + 5] = 0.0
    z[rows // 3] = z[rows // 3].round()
    z = z.to(dtype)
    if C > 2:
        hide = torch.rand(rows, C, generator=gen, device=dev) < 0.2
        z.masked_fill_(hide, -math.inf)
    z[1] = -math.inf
    z[rows - 2] = -math.inf
    z[rows - 2, C - 1] = 2.0
    z[rows - 3] = torch.finfo(dtype).min
    target = torch.randint(0, C, (rows,), generator=gen, device=dev)
    target[::17] = -100
    target[5] = C
    target[rows - 1] = -1
    z = strided(z, how)
    assert how == "plain" or z.stride(0) > C
    return z, target


KEPT = [0, 1, 2, 5, 10, 16, 32]


@pytest.mark.parametrize("C", [1, 2, 31, 32, 47, 64])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", ["plain", "wide", "odd"])
def test_many_short_rows(dev, C, dtype, how):
    """A lane a row (rows of at most 128 bytes), else four; gradient tiles of
    many rows."""
    rows = 70001
    assert rows >= 64 * 1024
    z, target = answers_of(dev, rows, C, dtype, how)
    for k in KEPT:
        if k <= C:
            check_answers(dev, z, target, k)


@pytest.mark.parametrize("C", [65, 100, 128, 129, 255, 256])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", ["plain", "wide", "odd"])
def test_many_rows_of_four_lanes(dev, C, dtype, how):
    """Four lanes a row: up to 512 bytes (above: sixteen)."""
    rows = 17001
    assert 4 * rows >= 64 * 1024
    z, target = answers_of(dev, rows, C, dtype, how)
    for k in KEPT:
        check_answers(dev, z, target, k)


@pytest.mark.parametrize("C", [1, 3, 47, 48, 300, 512, 700, 1024, 1365, 2047,
                               2048, 2049, 4096, 4097])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", ["plain", "wide", "odd"])
def test_gradient_tiles_of_several_rows(dev, C, dtype, how):
    """Gradient tiles that hold two rows, one, or part of one."""
    rows = 3001
    assert up(rows, 1024) > 1
    z, target = answers_of(dev, rows, C, dtype, how)
    for k in {0, min(C, 3), min(C, 32)}:
        check_answers(dev, z, target, k)


@pytest.mark.parametrize("dtype", TYPES)
def test_order_of_subnormal_logits(dev, dtype):
    """Values below the smallest normal one keep their order."""
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    for rows in (7, 70001):
        steps = torch.randint(-40, 40, (rows, 20), device=dev)
        z = (steps.double() * tiny).to(dtype)
        a = ops.log_probs(z, None, top_k=5)
        order = torch.sort(steps, dim=1, descending=True, stable=True).indices
        assert torch.equal(a.top_index, order[:, :5])


def test_no_rows(dev):
    for C in (1, 47, 5000, 20000):
        z = torch.zeros(0, C, device=dev, requires_grad=True)
        t = torch.zeros(0, dtype=torch.int64, device=dev)
        a = ops.log_probs(z, t, top_k=1)
        assert a.log_prob.shape == a.entropy.shape == (0,)
        assert a.top_index.shape == (0, 1)
        g, = torch.autograd.grad(a.log_prob.sum() + a.entropy.sum(), z)
        assert g.shape == z.shape


# ---------------------------------------------------------------------------
# the variants with workspaces, captured
# ---------------------------------------------------------------------------
def long_groups(dev):
    """The tiled plan, 256 x 256 products and dW by teams."""
    ids = torch.randint(-1, 6, (4400, 2), device=dev)
    x = torch.randn(4400, 2048, device=dev).bfloat16()
    w = (torch.randn(6, 2048, 2048, device=dev) / 45).bfloat16()

    def step(ids, x, w):
        route = ops.route_rows(ids, 6)
        xs = ops.dispatch_rows(route, x)
        y = ops.segment_mm(route.offsets, xs, w)
        out = ops.combine_rows(route, y)
        return (route.position, out) + torch.autograd.grad(
            out, (x, w), torch.ones_like(out))

    return [ids, x, w], step


def long_rows(dev):
    """Rows in parts that are joined."""
    z = torch.randn(9, 40001, device=dev).half()
    t = torch.randint(0, 40001, (9,), device=dev)

    def step(t, z):
        a = ops.log_probs(z, t, top_k=7)
        g, = torch.autograd.grad(a.log_prob.sum() + a.entropy.sum(), z)
        return a + (g,)

    return [t, z], step


@pytest.mark.parametrize("make", [long_groups, long_rows])
def test_workspaces_in_two_graphs(dev, make):
    """Two graphs of one program, replayed in turn with eager runs of it between
    and new inputs each time, give what the eager runs give."""
    ins, step = make(dev)

    def run(ts):
        return step(*[t.detach().requires_grad_(t.is_floating_point())
                      for t in ts])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run(ins)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(ins)
        graphs.append((graph, outs))
    for i in range(3):
        ins[0].copy_(ins[0].flip(0))
        ins[1].copy_(torch.randn(ins[1].shape, device=dev))
        want = run([t.clone() for t in ins])
        torch.cuda.synchronize()
        for graph, outs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
