"""The operators of the typed / mixture-of-experts path and of the classifier's
answer, as cases to measure: rows sorted by group and back (``route_rows``,
``dispatch_rows``, ``combine_rows``), the product of each group with its own
weight (``segment_mm``), and log probabilities with entropy and the best
alternatives (``log_probs``).

With ``own`` false, ``run`` computes them from elementary torch operations in
32 bits, rounded once at the end; with ``own`` true it makes the calls a user
makes. Sizes are those of this framework's workloads: batches of 1000 seeds
and the ~26.7K rows they sample, 100 features, 47 classes, 1345 relations,
14951 entities, embeddings of 400, and generic sizes around them.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a handful of rows answered at once: latency of the whole chain
        dict(name="route answer", op="route", rows=8, k=2, groups=8, width=256, type="bf16", train=False, pad=0.0),
        # the rows that one flagship batch samples, their 100 features sent to two experts each
        dict(name="route batch", op="route", rows=26752, k=2, groups=16, width=100, type="fp32", train=True, pad=0.0),
        # rows of embeddings sorted by relation, a tenth of the batch being padding
        dict(name="route relations", op="route", rows=65536, k=1, groups=1345, width=400, type="fp32", train=True, pad=0.1),
        # a full-graph layer with many experts
        dict(name="route layer", op="route", rows=262144, k=2, groups=64, width=512, type="bf16", train=True, pad=0.0),
        # eight rows on two experts each: reading the weights is all there is
        dict(name="mm answer", op="mm", rows=16, groups=8, k=256, n=512, type="bf16", train=False),
        # the input projection of a flagship batch, in the framework's default type
        dict(name="mm batch", op="mm", rows=53504, groups=16, k=100, n=256, type="fp32", train=True),
        # one matrix for each of many relations (the matrices are most of the bytes)
        dict(name="mm relations", op="mm", rows=65536, groups=1345, k=400, n=400, type="fp16", train=True),
        # a full-graph layer's experts: bound by the matrix cores
        dict(name="mm layer", op="mm", rows=262144, groups=8, k=512, n=1024, type="bf16", train=True),
        # tail entities for a few queries, known answers filtered out, the ten best
        dict(name="answer entities", op="answer", rows=8, classes=14951, top=10, type="fp32", train=False, masked=0.01),
        # the flagship's loss: 1000 seeds, 47 classes
        dict(name="answer batch", op="answer", rows=1000, classes=47, top=0, type="fp32", train=True, masked=0.0),
        # predictions for every node of a products-sized graph, with the five best
        dict(name="answer nodes", op="answer", rows=2449029, classes=47, top=5, type="fp16", train=False, masked=0.0),
        # a one-against-all loss over all entities, with the ten best kept
        dict(name="answer all", op="answer", rows=1024, classes=14951, top=10, type="bf16", train=True, masked=0.01),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("route", "mm", "answer"))
    kind, train = rng.choice(sorted(TYPES)), rng.random() < 0.6
    if op == "route":
        k, width = rng.randint(1, 4), _spread(rng, 16, 1024)
        most = 262144 * 2 * 512 // (k * width) // (2 if kind == "fp32" else 1)
        return dict(op=op, rows=_spread(rng, 1, min(most, 500000)), k=k, groups=_spread(rng, 2, 1345), width=width,
                    type=kind, train=train, pad=rng.choice((0.0, 0.0, 0.1, 0.5)))
    if op == "mm":
        k, n = _spread(rng, 16, 1024), _spread(rng, 16, 1024)
        most = 262144 * 512 * 1024 // (k * n) // (8 if kind == "fp32" else 1)
        groups = _spread(rng, 2, min(1345, 430_000_000 // (k * n)))
        return dict(op=op, rows=_spread(rng, 1, max(1, min(most, 200_000_000 // (k + n), 300000))), groups=groups, k=k, n=n, type=kind, train=train)
    classes = _spread(rng, 2, 200000)
    most = 2449029 * 47 // classes // (4 if train else 2 if kind == "fp32" else 1)
    return dict(op=op, rows=_spread(rng, 1, max(1, min(most, 2000000))), classes=classes, top=rng.randint(0, min(20, classes)),
                type=kind, train=train, masked=rng.choice((0.0, 0.0, 0.01, 0.3)))


# ---------------------------------------------------------------------------
# what a user has in hand before the call
# ---------------------------------------------------------------------------
def _normal(gen, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).to(dtype)


def _groups(gen, count, groups):
    """Group ids whose popularity falls as the square root of their rank, as relations' and experts' does."""
    share = torch.arange(1, groups + 1, device="cuda", dtype=torch.float32).rsqrt()
    share = share[torch.randperm(groups, generator=gen, device="cuda")]
    edges = torch.cumsum(share, 0)
    return torch.searchsorted(edges, torch.rand(count, generator=gen, device="cuda") * edges[-1]).clamp_(max=groups - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, train = TYPES[case["type"]], case["train"]
    state = dict(case)
    if case["op"] == "route":
        rows, k, width = case["rows"], case["k"], case["width"]
        ids = _groups(gen, rows * k, case["groups"]).view(rows, k)
        if case["pad"]:  # a padded row has no group in any of its slots
            ids[torch.rand(rows, generator=gen, device="cuda") < case["pad"]] = -1
        state["ids"] = ids
        state["x"] = _normal(gen, rows, width, dtype=dtype)
        state["y"] = _normal(gen, rows * k, width, dtype=dtype)  # what the experts made of the sorted rows
        state["weights"] = torch.softmax(torch.randn(rows, k, generator=gen, device="cuda"), 1)
        if train:
            state["grad_sorted"] = _normal(gen, rows * k, width, dtype=dtype)
            state["grad_out"] = _normal(gen, rows, width, dtype=dtype)
            for name in ("x", "y", "weights"):
                state[name].requires_grad_()
    elif case["op"] == "mm":
        rows, groups, k, n = case["rows"], case["groups"], case["k"], case["n"]
        count = torch.bincount(_groups(gen, rows, groups), minlength=groups)
        state["offsets"] = torch.zeros(groups + 1, dtype=torch.int64, device="cuda")
        torch.cumsum(count, 0, out=state["offsets"][1:])
        state["longest"] = int(count.max())  # a padded product needs it on the host
        state["x"] = _normal(gen, rows, k, dtype=dtype)
        state["weight"] = _normal(gen, groups, k, n, dtype=dtype, scale=k ** -0.5)
        if train:
            state["grad_out"] = _normal(gen, rows, n, dtype=dtype)
            state["x"].requires_grad_()
            state["weight"].requires_grad_()
    else:
        rows, classes = case["rows"], case["classes"]
        logits = _normal(gen, rows, classes, dtype=dtype, scale=3.0)
        state["target"] = torch.randint(0, classes, (rows,), generator=gen, device="cuda")
        if case["masked"]:  # filtered answers, the target never among them
            hide = torch.rand(rows, classes, generator=gen, device="cuda") < case["masked"]
            hide.scatter_(1, state["target"][:, None], False)
            logits.masked_fill_(hide, -math.inf)
        state["logits"] = logits
        if train:
            state["grad"] = tuple(torch.randn(rows, *tail, generator=gen, device="cuda") / rows for tail in ((), (), (case["top"],)))
            if case["masked"]:  # an alternative that the mask left without probability has no gradient
                left = (~hide).sum(1)
                keep = torch.arange(case["top"], device="cuda") < left[:, None]
                state["grad"] = state["grad"][:2] + (state["grad"][2] * keep,)
            state["logits"].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _own[state["op"]](state)
    with torch.no_grad():
        return _plain[state["op"]](state)


def _own_route(s):
    from dgl_operator_amd import ops

    route = ops.route_rows(s["ids"], s["groups"])
    xs = ops.dispatch_rows(route, s["x"])
    out = ops.combine_rows(route, s["y"], s["weights"])
    found = [route.offsets, route.position, xs, out]
    if s["train"]:
        found += torch.autograd.grad((xs, out), (s["x"], s["y"], s["weights"]), (s["grad_sorted"], s["grad_out"]))
    return found


def _own_mm(s):
    from dgl_operator_amd import ops

    y = ops.segment_mm(s["offsets"], s["x"], s["weight"])
    found = [y]
    if s["train"]:
        found += torch.autograd.grad(y, (s["x"], s["weight"]), s["grad_out"])
    return found


def _own_answer(s):
    from dgl_operator_amd import ops

    a = ops.log_probs(s["logits"], s["target"], top_k=s["top"])
    found = [a.log_prob, a.entropy, a.top_log_prob, a.top_index]
    if s["train"]:
        found += torch.autograd.grad(found[:3], s["logits"], s["grad"])
    return found


def _plain_route(s):
    ids, groups, x, y, w = s["ids"], s["groups"], s["x"], s["y"], s["weights"]
    rows, k = ids.shape
    slots = rows * k
    flat = ids.reshape(-1)
    kept = (flat >= 0) & (flat < groups)
    key = torch.where(kept, flat, groups)
    order = torch.argsort(key, stable=True)
    count = torch.zeros(groups + 1, dtype=torch.int64, device=x.device).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat((count.new_zeros(1), torch.cumsum(count[:groups], 0)))
    place = torch.empty_like(order)
    place[order] = torch.arange(slots, device=x.device)
    position = torch.where(kept, place, -1).view(rows, k).to(torch.int32)
    live = kept[order][:, None]
    xs = torch.where(live, x[order // k], 0)
    taken = torch.where(kept[:, None], y[place].float(), 0.0).view(rows, k, -1)
    out = (taken * w[:, :, None]).sum(1).to(y.dtype)
    found = [offsets, position, xs, out]
    if s["train"]:
        back = torch.where(kept[:, None], s["grad_sorted"][place].float(), 0.0).view(rows, k, -1)
        found.append(back.sum(1).to(x.dtype))
        g = s["grad_out"].float()
        scaled = (g[:, None, :] * w[:, :, None]).view(slots, -1).to(y.dtype)
        found.append(torch.where(live, scaled[order], 0))
        found.append((taken * g[:, None, :]).sum(2))
    return found


def _plain_mm(s):
    offsets, x, w = s["offsets"], s["x"], s["weight"]
    at = torch.arange(x.shape[0], device=x.device)
    group = torch.searchsorted(offsets, at, right=True) - 1
    slot = at - offsets[group]

    def padded(rows):
        out = torch.zeros(w.shape[0], s["longest"], rows.shape[1], device=x.device)
        out[group, slot] = rows.float()
        return out

    wide, w32 = padded(x), w.float()
    found = [torch.bmm(wide, w32)[group, slot].to(x.dtype)]
    if s["train"]:
        grad = padded(s["grad_out"])
        found.append(torch.bmm(grad, w32.transpose(1, 2))[group, slot].to(x.dtype))
        found.append(torch.bmm(wide.transpose(1, 2), grad).to(w.dtype))
    return found


def _plain_answer(s):
    z, t, top = s["logits"].float(), s["target"][:, None], s["top"]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    entropy = lse - torch.where(e > 0, e * z, 0.0).sum(1, keepdim=True) / total
    logp = z - lse
    found = [logp.gather(1, t)[:, 0], entropy[:, 0]]
    if top:
        index = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
    else:
        index = t[:, :0]
    found += [logp.gather(1, index), index]
    if s["train"]:
        g_lp, g_h, g_top = s["grad"]
        p = e / total
        pull = (g_lp + g_top.sum(1))[:, None] + g_h[:, None] * (torch.where(e > 0, logp, 0.0) + entropy)
        grad = (-p * pull).scatter_add_(1, t, g_lp[:, None]).scatter_add_(1, index, g_top)
        found.append(grad.to(s["logits"].dtype))
    return found


_own = {"route": _own_route, "mm": _own_mm, "answer": _own_answer}
_plain = {"route": _plain_route, "mm": _plain_mm, "answer": _plain_answer}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = TYPES[case["type"]].itemsize
    if case["op"] == "route":
        rows, k, width = case["rows"], case["k"], case["width"]
        slots = rows * k
        # ids, position, offsets, weights; x and out once, sorted rows and the experts' rows k times
        moved = 16 * slots + 8 * (case["groups"] + 1) + 2 * size * (rows + slots) * width
        done = 2 * slots * width
        if case["train"]:  # two gradients in, two out, and that of the weights
            moved += 2 * size * (rows + slots) * width + 4 * slots
            done *= 4
        return {"bytes": moved, "flops": done}
    if case["op"] == "mm":
        rows, k, n = case["rows"], case["k"], case["n"]
        moved = 8 * (case["groups"] + 1) + size * (rows * (k + n) + min(case["groups"], rows) * k * n)
        done = 2 * rows * k * n
        if case["train"]:
            moved += size * (rows * (k + n) + case["groups"] * k * n)
            done *= 3
        return {"bytes": moved, "flops": done}
    rows, classes, top = case["rows"], case["classes"], case["top"]
    moved = rows * (size * classes + 16 + 12 * top)
    done = 5 * rows * classes
    if case["train"]:
        moved += rows * (size * classes + 8 + 4 * top)
        done += 6 * rows * classes
    return {"bytes": moved, "flops": done}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    train = case["train"]
    if case["op"] == "mm":
        ends = s["offsets"].tolist()
        x, w = s["x"].double(), s["weight"].double()
        y = x.new_zeros(case["rows"], case["n"])
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        g = s["grad_out"].double() if train else None
        for i, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
            if a == b:
                continue
            y[a:b] = x[a:b].mm(w[i])
            if train:
                dx[a:b] = g[a:b].mm(w[i].t())
                dw[i] = x[a:b].t().mm(g[a:b])
        return [y, dx, dw] if train else [y]
    if case["op"] == "route":
        rows, k, width, slots = case["rows"], case["k"], case["width"], case["rows"] * case["k"]
        flat = s["ids"].reshape(-1)
        live = (flat >= 0).nonzero()[:, 0]
        # slots of one group follow each other in their own order
        live = live[torch.sort(flat[live] * slots + live).indices]
        token = live // k
        many = len(live)
        x, y, w = s["x"].double(), s["y"].double()[:many], s["weights"].double().reshape(-1)[live]
        xs, out = x.new_zeros(slots, width), x.new_zeros(rows, width)
        xs[:many] = x[token]
        out.index_add_(0, token, y * w[:, None])
        found = [None, None, xs, out]
        if train:
            g = s["grad_out"].double()[token]
            dx, dy, dw = torch.zeros_like(x), x.new_zeros(slots, width), x.new_zeros(slots)
            dx.index_add_(0, token, s["grad_sorted"].double()[:many])
            dy[:many] = g * w[:, None]
            dw[live] = (g * y).sum(1)
            found += [dx, dy, dw.view(rows, k)]
        return found
    z, t, top = s["logits"].double(), s["target"], case["top"]
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    entropy = -torch.xlogy(p, p).sum(1)
    best = logp.topk(top, 1).values if top else logp[:, :0]
    found = [logp[torch.arange(case["rows"], device=z.device), t], entropy, best, None]
    if train:
        index = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]  # of equal logits the first
        g_lp, g_h, g_top = (v.double() for v in s["grad"])
        # each answer's Jacobian row is its unit vector less p; the entropy's is -p (log p + H)
        grad = -p * (g_lp + g_top.sum(1))[:, None] - g_h[:, None] * (torch.xlogy(p, p) + p * entropy[:, None])
        grad[torch.arange(case["rows"], device=z.device), t] += g_lp
        grad.scatter_add_(1, index, g_top)
        found.append(grad)
    return found
