"""Workloads of the adapter and gradient operators, for timing and for checking their outputs.

Three groups of calls: rows sorted by adapter (`group_rows`), a shared projection with low-rank adapters and its backward
pass (`adapter_linear`, `adapter_linear_backward`), and the global gradient norm with clipping (`clip_grad_norm_`).
`listed()` names fixed cases, `draw()` makes more of the same ranges, `run()` is one pass through a case: in plain torch
operations, or, with `own` set, through the package."""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
LARGEST = 16384 * 4096 * 4096                        # rows * in * out of the largest projection below
LARGEST_CLIP = 1 << 28                               # elements of the largest set of gradients below


# ---- cases -----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one rollout step of a few environments: the agents that ask for a decision, 20 maps with an adapter each
        dict(name="group-step", op="group", rows=317, adapters=20, spread="runs", bare=0.0),
        # a large rollout step: every row of thousands of environments, one adapter per environment
        dict(name="group-wide", op="group", rows=262144, adapters=1024, spread="random", bare=0.05),
        # acting for one agent: the first dense layer of a network of 70 rails (64 filters * 3 planes * 70 rails -> 512)
        dict(name="act-one", op="forward", type="float32", rows=1, inputs=13440, outputs=512, rank=16, adapters=20,
             spread="random", bare=0.0, bias=True, features="relu"),
        # single tokens of 37 requests that use 24 adapters between them
        dict(name="serve-37", op="forward", type="bfloat16", rows=37, inputs=4096, outputs=4096, rank=16, adapters=24,
             spread="random", bare=0.1, bias=False, features="normal"),
        # a replay sample of 512 transitions from 20 maps, the same dense layer
        dict(name="learn-512", op="forward", type="float32", rows=512, inputs=13440, outputs=512, rank=16, adapters=20,
             spread="random", bare=0.0, bias=True, features="relu"),
        # sizes that are a multiple of nothing
        dict(name="odd-1001", op="forward", type="float16", rows=1001, inputs=1003, outputs=515, rank=5, adapters=7,
             spread="skewed", bare=0.2, bias=True, features="normal"),
        # a long mixed batch of a wide layer, the largest product
        dict(name="batch-16k", op="forward", type="bfloat16", rows=16384, inputs=4096, outputs=4096, rank=64, adapters=48,
             spread="skewed", bare=0.05, bias=True, features="normal"),
        # gradients of the adapters alone for a replay sample: the shared layer and what feeds it stay as they are
        dict(name="learn-512-back", op="backward", type="float32", rows=512, inputs=13440, outputs=512, rank=16,
             adapters=20, spread="random", bare=0.0, features="relu", dx=False),
        # the backward pass in the middle of a network: the gradient of the inputs as well
        dict(name="batch-4k-back", op="backward", type="bfloat16", rows=4099, inputs=4096, outputs=4096, rank=32,
             adapters=24, spread="skewed", bare=0.05, features="normal", dx=True),
        # the gradient tensors of one small network: ten tensors, mostly biases
        dict(name="clip-small", op="clip", type="float32", tensors=10, elements=60000, max_norm=1.0),
        # the gradient of a network of 70 rails: two weight blocks hold nearly all of it
        dict(name="clip-network", op="clip", type="float32", tensors=10, elements=13789635, max_norm=10.0),
        # many tensors of a large model
        dict(name="clip-many", op="clip", type="bfloat16", tensors=291, elements=LARGEST_CLIP, max_norm=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["group", "forward", "forward", "forward", "backward", "backward", "clip"])
    spread = rng.choice(["random", "skewed", "runs"])
    bare = rng.choice([0.0, 0.05, 0.2])
    if op == "group":
        return dict(op=op, rows=_log(rng, 1, 262144), adapters=_log(rng, 1, 1024), spread=spread, bare=bare)
    kind = rng.choice(["float32", "bfloat16", "float16"])
    if op == "clip":
        tensors = _log(rng, 1, 300)
        return dict(op=op, type=kind, tensors=tensors, elements=_log(rng, max(1000, 2 * tensors), LARGEST_CLIP // 2),
                    max_norm=rng.choice([0.5, 1.0, 10.0]))
    while True:
        rows, inputs, outputs = _log(rng, 1, 16384), _log(rng, 64, 13440), _log(rng, 32, 8192)
        if rng.random() < 0.6:                       # most layers have whole multiples of 64 inputs and outputs
            inputs, outputs = -(-inputs // 64) * 64, -(-outputs // 64) * 64
        if rows * inputs * outputs <= LARGEST // (8 if kind == "float32" else 2):
            break
    case = dict(op=op, type=kind, rows=rows, inputs=inputs, outputs=outputs, rank=_log(rng, 1, 128),
                adapters=_log(rng, 1, 64), spread=spread, bare=bare, features=rng.choice(["normal", "relu"]))
    if op == "forward":
        case["bias"] = rng.random() < 0.5
    else:
        case["dx"] = rng.random() < 0.5
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _ids(case, gen):
    """Which adapter every row uses (-1: none), on the host: a user's program knows who asked."""
    n, e = case["rows"], case["adapters"]
    if case["spread"] == "skewed":                   # a few adapters have most of the rows
        ids = (torch.rand(n, generator=gen) ** 3 * e).long().clamp_(max=e - 1)
    else:
        ids = torch.randint(0, e, (n,), generator=gen)
    if case["spread"] == "runs":                     # two ascending runs: departing agents, then agents at a switch
        cut = n // 3
        ids = torch.cat([ids[:cut].sort().values, ids[cut:].sort().values])
    ids[torch.rand(n, generator=gen) < case["bare"]] = -1
    return ids


def _tensor_sizes(case):
    """Sizes of the gradient tensors: half of them small (biases, norms), the others share the rest unevenly."""
    count, total = case["tensors"], case["elements"]
    gen = torch.Generator().manual_seed(count)
    if count == 1:
        return [total]
    small = count // 2
    budget = max(1, total // (50 * count))
    sizes = [1 + int(x) for x in torch.randint(0, budget, (small,), generator=gen)]
    parts = torch.rand(count - small, generator=gen) + 0.1
    rest = total - sum(sizes)
    sizes += [max(1, int(rest * float(p / parts.sum()))) for p in parts]
    sizes[-1] += max(0, total - sum(sizes))
    order = torch.randperm(count, generator=gen).tolist()
    return [sizes[i] for i in order]


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * scale

    state = {"case": case}
    if case["op"] == "clip":
        # the tensors are pieces of one buffer, as an optimizer over flat buffers keeps them; the clipped gradients go
        # into the pieces of another
        sizes = _tensor_sizes(case)
        state["flat"] = normal(sum(sizes), scale=0.02).to(TYPES[case["type"]])
        state["clipped"] = torch.empty_like(state["flat"])
        state["grads"] = list(state["flat"].split(sizes))
        state["out"] = list(state["clipped"].split(sizes))
        return state
    ids = _ids(case, host)
    state["ids"] = ids.to(torch.int32).cuda()
    if case["op"] == "group":
        return state
    e = case["adapters"]
    state["counts"] = torch.bincount(ids[ids >= 0], minlength=e).tolist()
    kind = TYPES[case["type"]]
    k, n_out, r, rows = case["inputs"], case["outputs"], case["rank"], case["rows"]
    x = normal(rows, k)
    state["x"] = (x.relu_() if case["features"] == "relu" else x).to(kind)
    state["weight"] = normal(n_out, k, scale=k ** -0.5).to(kind)
    state["a"] = normal(e, r, k, scale=k ** -0.5).to(kind)
    state["b"] = normal(e, n_out, r, scale=r ** -0.5).to(kind)
    state["scale"] = (0.25 + 1.75 * torch.rand(e, generator=host)).cuda()
    if case["op"] == "forward":
        state["bias"] = normal(n_out, scale=0.1).to(kind) if case["bias"] else None
        return state
    state["dy"] = normal(rows, n_out, scale=rows ** -0.5).to(kind)
    # what the forward pass kept: A x of every row
    low = torch.zeros(rows, r, device="cuda")
    order = torch.argsort(torch.where(ids < 0, e, ids), stable=True).cuda()
    lo = 0
    for i, count in enumerate(state["counts"]):
        if count:
            pick = order[lo:lo + count]
            low[pick] = state["x"][pick].float() @ state["a"][i].float().t()
        lo += count
    state["low"] = low
    if own:                                          # ... and the rows' order
        from flatland_marl_amd.adapters import group_rows
        state["groups"] = group_rows(state["ids"], e)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    case = state["case"]
    if case["op"] == "clip":
        from flatland_marl_amd.gradients import clip_grad_norm_
        norm = clip_grad_norm_(state["grads"], case["max_norm"], out=state["out"])
        return [norm, state["clipped"]]
    from flatland_marl_amd import adapters
    if case["op"] == "group":
        groups = adapters.group_rows(state["ids"], case["adapters"])
        return [groups.order, groups.offsets]
    if case["op"] == "forward":
        groups = adapters.group_rows(state["ids"], case["adapters"])
        return adapters.adapter_linear(state["x"], state["weight"], state["bias"], state["a"], state["b"], groups,
                                       scale=state["scale"])
    dx, da, db = adapters.adapter_linear_backward(state["dy"], state["x"], state["weight"], state["a"], state["b"],
                                                  state["groups"], state["low"], scale=state["scale"],
                                                  need_dx=case["dx"])
    return [dx, da, db] if case["dx"] else [da, db]


def _sorted_rows(ids, adapters):
    key = torch.where((ids >= 0) & (ids < adapters), ids, adapters)
    order = torch.argsort(key, stable=True)
    bounds = torch.arange(adapters + 1, device=ids.device, dtype=key.dtype)
    return order, torch.searchsorted(key[order], bounds)


def _run_plain(state):
    case = state["case"]
    if case["op"] == "clip":
        total = torch.zeros((), device="cuda")
        for g in state["grads"]:
            g = g.float()
            total = total + (g * g).sum()
        norm = total.sqrt()
        factor = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        for g, out in zip(state["grads"], state["out"]):
            out.copy_(g.float() * factor)
        return [norm, state["clipped"]]
    order, offsets = _sorted_rows(state["ids"], case["adapters"])
    if case["op"] == "group":
        return [order.to(torch.int32), offsets.to(torch.int32)]
    kind = state["x"].dtype
    x, weight = state["x"].float(), state["weight"].float()
    a, b, scale = state["a"].float(), state["b"].float(), state["scale"]
    if case["op"] == "forward":
        y = x @ weight.t()
        if state["bias"] is not None:
            y = y + state["bias"].float()
        lo = 0
        for i, count in enumerate(state["counts"]):
            if count:
                pick = order[lo:lo + count]
                y[pick] += ((x[pick] @ a[i].t()) @ b[i].t()) * scale[i]
            lo += count
        return y.to(kind)
    dy = state["dy"].float()
    dx = dy @ weight if case["dx"] else None
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    lo = 0
    for i, count in enumerate(state["counts"]):
        if count:
            pick = order[lo:lo + count]
            rows = dy[pick] * scale[i]
            u = rows @ b[i]
            da[i] = u.t() @ x[pick]
            db[i] = rows.t() @ state["low"][pick]
            if dx is not None:
                dx[pick] += u @ a[i]
        lo += count
    out = [da.to(kind), db.to(kind)]
    return out if dx is None else [dx.to(kind)] + out


# ---- what a pass cannot do without, and what it should give -----------------------------------------------------------
def work(case):
    if case["op"] == "group":
        return {"bytes": 8 * case["rows"] + 4 * (case["adapters"] + 1), "flops": case["rows"]}
    size = SIZE[case["type"]]
    if case["op"] == "clip":
        return {"bytes": 2 * size * case["elements"], "flops": 3 * case["elements"]}
    n, k, n_out, r = case["rows"], case["inputs"], case["outputs"], case["rank"]
    used = min(case["adapters"], n)
    if case["op"] == "forward":
        return {"bytes": size * (n * k + n_out * k + n * n_out + (n_out if case["bias"] else 0) + used * r * (k + n_out)),
                "flops": 2 * n * k * n_out + 2 * n * r * (k + n_out)}
    # without dx neither the weight nor A is read
    values = n * n_out + n * k + used * r * n_out + case["adapters"] * r * (k + n_out)
    flops = 2 * n * r * (n_out + n_out + k)
    if case["dx"]:
        values += n_out * k + n * k + used * r * k
        flops += 2 * n * k * n_out + 2 * n * r * k
    return {"bytes": size * values + 4 * n * r, "flops": flops}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "clip":
        flat = state["flat"].double()
        norm = math.sqrt(float(flat.square().sum()))
        factor = min(1.0, case["max_norm"] / (norm + 1e-6))
        return [torch.tensor(norm, dtype=torch.float64, device="cuda"), flat * factor]
    ids = state["ids"].tolist()
    members = [[] for _ in range(case["adapters"])]
    bare = []
    for row, e in enumerate(ids):
        (members[e] if 0 <= e < case["adapters"] else bare).append(row)
    if case["op"] == "group":
        flat, offsets = [], [0]
        for rows in members:
            flat += rows
            offsets.append(len(flat))
        return [torch.tensor(flat + bare, dtype=torch.int32, device="cuda"),
                torch.tensor(offsets, dtype=torch.int32, device="cuda")]
    x, w = state["x"].double(), state["weight"].double()
    if case["op"] == "forward":
        y = torch.matmul(x, w.transpose(0, 1).contiguous())
        if state["bias"] is not None:
            y += state["bias"].double()
        for e, rows in enumerate(members):
            if rows:
                pick = torch.tensor(rows, device="cuda")
                product = torch.matmul(state["b"][e].double(), state["a"][e].double())       # [outputs, inputs]
                y[pick] += float(state["scale"][e]) * torch.matmul(x[pick], product.t().contiguous())
        return y
    dy, low = state["dy"].double(), state["low"].double()
    dx = torch.matmul(dy, w) if case["dx"] else None
    da = torch.zeros_like(state["a"], dtype=torch.float64)
    db = torch.zeros_like(state["b"], dtype=torch.float64)
    for e, rows in enumerate(members):
        if not rows:
            continue
        pick = torch.tensor(rows, device="cuda")
        s = float(state["scale"][e])
        u = s * torch.matmul(dy[pick], state["b"][e].double())
        da[e] = torch.matmul(u.t().contiguous(), x[pick])
        db[e] = s * torch.matmul(dy[pick].t().contiguous(), low[pick])
        if dx is not None:
            dx[pick] += torch.matmul(u, state["a"][e].double())
    return [da, db] if dx is None else [dx, da, db]
