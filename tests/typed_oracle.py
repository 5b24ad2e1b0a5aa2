"""Oracles in 64 bits, and the error bounds, of the typed-row operators.

Bounds count roundings: `half(t)` is the largest relative error of one rounding
to type t; U = 2^-24 is that of fp32, in which the operators sum. A matrix
instruction may truncate where a vector one rounds, so its sums count 2 U a step.
"""
import math

import torch

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest step (subnormals), for results next to zero."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps


def route(ids, groups):
    """offsets, position, source by a plain loop."""
    ids = ids.reshape(-1).tolist()
    buckets = [[] for _ in range(groups)]
    for f, g in enumerate(ids):
        if 0 <= g < groups:
            buckets[g].append(f)
    offsets, source, position = [0], [], [-1] * len(ids)
    for b in buckets:
        for f in b:
            position[f] = len(source)
            source.append(f)
        offsets.append(len(source))
    source += [-1] * (len(ids) - len(source))
    return (torch.tensor(offsets), torch.tensor(position, dtype=torch.int32),
            torch.tensor(source, dtype=torch.int32))


def dispatch(x, position):
    k = position.shape[1]
    out = x.new_zeros((position.numel(), x.shape[1]))
    for f, p in enumerate(position.reshape(-1).tolist()):
        if p >= 0:
            out[p] = x[f // k]
    return out


def taken(y, position):
    flat = position.reshape(-1).long()
    rows = y.double()[flat.clamp(min=0)] if y.shape[0] else \
        y.new_zeros((flat.numel(), y.shape[1])).double()
    rows = torch.where(flat[:, None] >= 0, rows, 0.0)
    return rows.view(*position.shape, y.shape[1])


def combine(y, position, weights):
    """(result, bound): k products and sums in fp32, one rounding."""
    t = taken(y, position)
    w = torch.ones(position.shape, dtype=torch.float64) if weights is None \
        else weights.double()
    terms = t * w[:, :, None]
    ref, size = terms.sum(1), terms.abs().sum(1)
    k = position.shape[1]
    acc = (2 * k + 1) * U * size
    return ref, acc + half(y.dtype) * (ref.abs() + acc) + tiny(y.dtype)


def matmul(a, b, dtype, factor=2):
    """(a @ b in 64 bits, bound) for a sum of a.shape[-1] products in fp32."""
    a, b = a.double(), b.double()
    ref, size = a @ b, a.abs() @ b.abs()
    acc = factor * (a.shape[-1] + 2) * U * size
    return ref, acc + half(dtype) * (ref.abs() + acc) + tiny(dtype)


def segments(offsets):
    o = offsets.tolist()
    return list(enumerate(zip(o[:-1], o[1:])))


def segment_mm(offsets, x, w):
    ref = torch.zeros((x.shape[0], w.shape[2]), dtype=torch.float64)
    tol = torch.full_like(ref, 0.0)
    for g, (a, b) in segments(offsets):
        ref[a:b], tol[a:b] = matmul(x[a:b], w[g], x.dtype)
    return ref, tol


def segment_wgrad(offsets, x, grad):
    ref = torch.zeros((offsets.numel() - 1, x.shape[1], grad.shape[1]),
                      dtype=torch.float64)
    tol = torch.zeros_like(ref)
    for g, (a, b) in segments(offsets):
        if b > a:
            ref[g], tol[g] = matmul(x[a:b].t(), grad[a:b], x.dtype)
    return ref, tol


def log_probs(z, target, k, ignore=-100):
    """lp, entropy, top, index in 64 bits, row by row."""
    z = z.double()
    n, C = z.shape
    lp, ent = torch.empty(n).double(), torch.empty(n).double()
    top, index = torch.empty(n, k).double(), torch.empty(n, k).long()
    full = torch.empty_like(z)
    for r in range(n):
        row = z[r]
        if bool((row == -math.inf).all()):
            logp, ent[r] = row.clone(), 0.0
        else:
            logp = torch.log_softmax(row, 0)
            p = logp.exp()
            ent[r] = -torch.xlogy(p, p).sum()
        full[r] = logp
        order = sorted(range(C), key=lambda j: (
            0 if math.isnan(row[j]) else 1,
            0.0 if math.isnan(row[j]) else -float(row[j]), j)) if k else []
        index[r] = torch.tensor(order[:k], dtype=torch.long)
        top[r] = logp[index[r]]
        t = None if target is None else int(target[r])
        lp[r] = 0.0 if t is None or t == ignore else \
            logp[t] if 0 <= t < C else math.nan
    return lp, ent, top, index, full


def log_probs_grad(z, target, index, logp, ent, g_lp, g_ent, g_top, ignore=-100):
    n, C = z.shape
    p = logp.exp()
    grad = torch.zeros(n, C).double()
    pull = torch.zeros(n).double()
    rows = torch.arange(n)
    if g_lp is not None:
        g = g_lp.double().clone()
        g[target == ignore] = 0.0
        g[(target != ignore) & ((target < 0) | (target >= C))] = math.nan
        grad[rows, target.clamp(0, C - 1)] += torch.nan_to_num(g)
        pull += g
    if g_top is not None:
        grad.scatter_add_(1, index, g_top.double())
        pull += g_top.double().sum(1)
    grad -= p * pull[:, None]
    if g_ent is not None:
        grad -= g_ent.double()[:, None] * (
            torch.xlogy(p, p) + p * ent[:, None])
    grad[(z == -math.inf).all(1)] = 0.0
    return grad


def log_s_error(z):
    """How far log(sum e^(z - m)) may be off, per row: the rounding of each
    (z - m) acts on its e^(z - m) (times |z - m| U, at most |x| e^-|x| < 0.4
    weighted), four roundings in each exponential, and at most C / 64 + 272
    additions on the way of any term to the sum; the entropy's sum has one
    product more and |z - m| as a factor of its terms."""
    C = z.shape[1]
    steps = min(C, C // 64 + 256) + 16
    return (steps + 8) * U
