"""Plain 64-bit forms of the adapter operators on the CPU, with bounds for the kernels' rounding."""
import torch


def rand(seed, *shape, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale


def case(seed, n, k, n_out, r, e, kind, bare=0.2, skew=False):
    """Inputs as the type holds them: dict of CPU tensors (x, weight, bias, a, b, dy of `kind`; scale float32; ids int32)."""
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand(n, generator=g) ** (3 if skew else 1) * e).long().clamp_(max=e - 1)
    ids[torch.rand(n, generator=g) < bare] = -1
    c = dict(x=rand(seed + 1, n, k), weight=rand(seed + 2, n_out, k, scale=k ** -0.5), bias=rand(seed + 3, n_out),
             a=rand(seed + 4, e, r, k, scale=k ** -0.5), b=rand(seed + 5, e, n_out, r, scale=r ** -0.5),
             dy=rand(seed + 6, n, n_out, scale=n ** -0.5))
    c = {name: t.to(kind) for name, t in c.items()}
    c["scale"] = 0.25 + torch.rand(e, generator=g)
    c["ids"] = ids.to(torch.int32)
    return c


def _members(c):
    return [(e, (c["ids"] == e).nonzero().flatten()) for e in range(c["a"].shape[0])]


def forward(c, absolute=False):
    """(y, low) in 64 bits; absolute: of the absolute values (what rounding errors are relative to)."""
    f = (lambda t: t.double().abs()) if absolute else (lambda t: t.double())
    x, y = f(c["x"]), f(c["x"]) @ f(c["weight"]).t() + f(c["bias"])
    low = torch.zeros(x.shape[0], c["a"].shape[1], dtype=torch.float64)
    for e, rows in _members(c):
        if len(rows):
            low[rows] = x[rows] @ f(c["a"][e]).t()
            y[rows] += float(c["scale"][e]) * (low[rows] @ f(c["b"][e]).t())
    return y, low


def backward(c, low, absolute=False):
    """(dx, da, db) in 64 bits for low as given."""
    f = (lambda t: t.double().abs()) if absolute else (lambda t: t.double())
    x, dy, low = f(c["x"]), f(c["dy"]), f(low)
    dx = dy @ f(c["weight"])
    da, db = torch.zeros(c["a"].shape, dtype=torch.float64), torch.zeros(c["b"].shape, dtype=torch.float64)
    for e, rows in _members(c):
        if len(rows):
            s = float(c["scale"][e])
            u = s * (dy[rows] @ f(c["b"][e]))
            dx[rows] += u @ f(c["a"][e])
            da[e] = u.t() @ x[rows]
            db[e] = s * (dy[rows].t() @ low[rows])
    return dx, da, db


def bound(exact, absolute, terms, kind):
    """Largest error of a result.  Sums are kept in fp32: one rounding (2^-24 of at most the sum of absolute values) per
    matrix instruction and 16 elements of the sum, six instructions where fp32 operands are split in three; about 64 more
    for trees inside an instruction, slices that are added up and the second of two chained sums.  bf16 and fp16 results:
    the narrow intermediate is held to 2^-17 in the product behind it (twice that for a value just below a power of two),
    and the result is rounded once, by half a step."""
    c = (6 * terms / 16 + 64) * 2.0 ** -24
    if kind != torch.float32:
        c = (terms / 16 + 64) * 2.0 ** -24 + 2.0 ** -16
    step = torch.finfo(kind).eps / 2
    tiny = torch.finfo(kind).smallest_normal * torch.finfo(kind).eps       # half the smallest step there is
    return c * absolute * (1 + step) + step * exact.abs() + tiny


def to_gpu(c):
    return {name: t.cuda() for name, t in c.items()}
