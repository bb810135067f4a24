"""The adapter operators on values at the ends of their types, against plain 64-bit forms.  Needs an MI355X."""
import pytest
import torch

from tests import adapter_ref as ref

pytestmark = pytest.mark.gpu
ROWS = [1, 24, 64, 65, 150]                                  # few-row form, its last size, tiles
TOP = torch.finfo(torch.float32).max


def _check(got, exact, absolute, terms, kind):
    assert torch.isfinite(got).all()
    err = (got.cpu().double() - exact).abs()
    worst = (err / ref.bound(exact, absolute, terms, kind)).max().item()
    assert worst <= 1.0, worst


def _small(n, k, n_out, r, e, kind, seed):
    """A case whose operands are all around 2^-6, with every row on adapter 0 or 1."""
    c = ref.case(seed, n, k, n_out, r, e, kind, bare=0.0)
    for name in ("x", "weight", "bias", "a", "b", "dy"):
        c[name] = (c[name].double() / c[name].double().abs().max() * 2.0 ** -6).to(kind)
    c["ids"] = torch.arange(n, dtype=torch.int32) % 2
    return c


def _both_passes(c, low=None):
    from flatland_marl_amd.adapters import adapter_linear, adapter_linear_backward, group_rows
    n, k = c["x"].shape
    n_out, r = c["b"].shape[1:]
    kind = c["x"].dtype
    d = ref.to_gpu(c)
    g = group_rows(d["ids"], c["a"].shape[0])
    y, kept = adapter_linear(d["x"], d["weight"], d["bias"], d["a"], d["b"], g, scale=d["scale"], keep_low=True)
    # (what errors are relative to: the sum of the products' absolute values, so the factor's absolute value as well)
    whole = dict(c, scale=c["scale"].abs())
    (want, want_low), (size, size_low) = ref.forward(c), ref.forward(whole, absolute=True)
    _check(kept, want_low, size_low, k, torch.float32)
    _check(y, want, size, k + r, kind)
    low = want_low.float() if low is None else low
    got = adapter_linear_backward(d["dy"], d["x"], d["weight"], d["a"], d["b"], g, low.cuda(), scale=d["scale"])
    for t, w, s, terms in zip(got, ref.backward(c, low), ref.backward(whole, low, absolute=True), (n_out + r, n_out + n, n)):
        _check(t, w, s, terms, kind)


@pytest.mark.parametrize("r", [5, 16])
@pytest.mark.parametrize("where", ["x", "weight", "a", "b", "dy"])
@pytest.mark.parametrize("n", ROWS)
def test_largest_finite_values(n, where, r):
    """The largest and the lowest value that fp32 has, in one operand at a time: no result is infinite by the formula."""
    c = _small(n, 72, 56, r, 2, torch.float32, 3)
    t = c[where]
    flat = t.view(-1)
    flat[::37] = TOP
    flat[5::41] = -TOP
    # (sums of a few products of 5e36 each stay below 3.4e38; so do those that pass through a second operand of 2^-6)
    _both_passes(c)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n", ROWS)
def test_narrow_products_above_the_largest_bf16(n, kind):
    """low = A x between the largest bf16 and the largest fp32; u = s B^T dy as well."""
    c = _small(n, 40, 56, 9, 2, kind, 7)
    top = torch.finfo(torch.bfloat16).max
    c["scale"].fill_(1.0)
    for wide, narrow in (("x", "a"), ("dy", "b")):
        c[wide][:, :2] = torch.tensor([top, 2.0 ** 119 * 1.875], dtype=torch.float64).to(kind)
        if wide == "x":
            c[narrow][:, 0] = 0.0
            c[narrow][:, 0, :2] = 1.0
        else:
            c[narrow][:, :, 0] = 0.0
            c[narrow][:, :2, 0] = 1.0
        c["weight"][:, :2] = 0.0
        c["weight"][:2] = 0.0
        low = ref.forward(c)[1]
        if wide == "x":
            assert (low[:, 0] > top).all() and (low[:, 0] <= TOP).all()
            c["b"][:, :, 0] = 2.0 ** -7
            _both_passes(c)
        else:
            c["x"] = c["x"].double().clamp(-2.0 ** -6, 2.0 ** -6).to(kind)
            c["a"][:, 0] = 2.0 ** -7
            # dA: sums over up to n / 2 + 1 rows of u x
            c["x"] = (c["x"].double() / n).to(kind)
            _both_passes(c)
    # low as the caller hands it over
    c = _small(n, 40, 56, 9, 2, kind, 8)
    low = ref.forward(c)[1].float()
    low[::5, 3] = TOP
    low[1::7, 8] = -TOP
    c["dy"] = (c["dy"].double() / n).to(kind)
    _both_passes(c, low)


@pytest.mark.parametrize("scale", [3.0, -200.0, 2.0 ** -20])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n", ROWS)
def test_scaled_narrow_products_outside_the_range(n, kind, scale):
    """low or u of 1.5e38: the factor takes them, or a sum without the factor is, beyond fp32; no result is."""
    big = 2.0 ** 126 * 1.75
    met = 2.0 ** -16 if abs(scale) > 1 else 4.0              # what the large one is multiplied with
    for large in ("x", "dy"):
        c = _small(n, 40, 56, 9, 2, kind, 11)
        c["scale"].fill_(scale)
        for name in ("a", "b", "x", "dy"):
            c[name] = (c[name].double() * 2.0 ** -10).to(kind)
        c[large][:, 0] = big
        if large == "x":                                     # low[:, 0] = x[:, 0], the other ranks do not see it
            c["a"][:, :, 0], c["a"][:, 0, 1:], c["a"][:, 0, 0] = 0.0, 0.0, 1.0
            c["weight"][:, 0] = 0.0
            c["b"][:, :, 0] = met
            c["dy"][:, 0] = met
        else:                                                # u[:, 0] = scale * dy[:, 0]
            c["b"][:, 0], c["b"][:, 1:, 0], c["b"][:, 0, 0] = 0.0, 0.0, 1.0
            c["weight"][0] = 0.0
            c["a"][:, 0] = met
            c["x"][:, 0] = met
        _both_passes(c)


def _same_places(got, exact, absolute, terms, kind):
    """Not finite exactly where the formula is not; NaN or that infinity there, and within the bound elsewhere."""
    got = got.cpu().double()
    bad = ~torch.isfinite(exact)
    assert torch.equal(~torch.isfinite(got), bad)
    infinite = torch.isinf(got)
    assert torch.equal(got[infinite], exact[infinite])
    tol = ref.bound(exact, absolute, terms, kind)
    assert ((got - exact).abs() <= tol)[~bad].all()


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("where", ["x", "weight", "bias", "a", "b", "dy", "low"])
@pytest.mark.parametrize("n", ROWS)
def test_infinities_are_not_lost_and_reach_no_other_sum(n, where, kind):
    """An infinity of either sign and a NaN in one operand at a time, among operands some of whose bf16 terms are zero."""
    from flatland_marl_amd.adapters import adapter_linear, adapter_linear_backward, group_rows
    k, n_out, r, e = 72, 56, 9, 4
    c = ref.case(17, n, k, n_out, r, e, kind, bare=0.0)
    c["ids"] = torch.arange(n, dtype=torch.int32) % e
    c["a"][2], c["b"][3] = (c[m][i].double().mul(8).round().div(8).to(kind) for m, i in (("a", 2), ("b", 3)))
    low = ref.forward(c)[1].float()
    t = low if where == "low" else c[where]
    flat = t.view(-1)
    for i, bad in enumerate((float("inf"), -float("inf"), float("nan"))):
        flat[(i * 31 + 5) % flat.numel()] = bad
    d = ref.to_gpu(c)
    g = group_rows(d["ids"], e)
    y, kept = adapter_linear(d["x"], d["weight"], d["bias"], d["a"], d["b"], g, scale=d["scale"], keep_low=True)
    got = adapter_linear_backward(d["dy"], d["x"], d["weight"], d["a"], d["b"], g, low.cuda(), scale=d["scale"])
    finite = {name: t.double().nan_to_num(0.0, 0.0, 0.0) if t.is_floating_point() else t for name, t in c.items()}
    (want, want_low), (size, size_low) = ref.forward(c), ref.forward(finite, absolute=True)
    _same_places(kept, want_low, size_low, k, torch.float32)
    _same_places(y, want, size, k + r, kind)
    sizes = ref.backward(finite, low.double().nan_to_num(0.0, 0.0, 0.0), absolute=True)
    for t, w, s, terms in zip(got, ref.backward(c, low), sizes, (n_out + r, n_out + n, n)):
        _same_places(t, w, s, terms, kind)


@pytest.mark.parametrize("power", [-100, -112, -120, -124])
@pytest.mark.parametrize("n", ROWS)
def test_small_fp32_values_are_held_to_the_smallest_bf16(n, power):
    """x and dy of 2^power: each enters its products, and so do low and u, with an error of at most 2^-133 beside fp32's."""
    from flatland_marl_amd.adapters import adapter_linear, adapter_linear_backward, group_rows
    k, n_out, r, e = 72, 56, 9, 4
    c = ref.case(31, n, k, n_out, r, e, torch.float32, bare=0.0)
    for name in ("x", "dy"):
        c[name] = (c[name].double() * 2.0 ** power).float()
    c["bias"].zero_()
    low = ref.forward(c)[1].float()
    d = ref.to_gpu(c)
    g = group_rows(d["ids"], e)
    y, kept = adapter_linear(d["x"], d["weight"], d["bias"], d["a"], d["b"], g, scale=d["scale"], keep_low=True)
    dx = adapter_linear_backward(d["dy"], d["x"], d["weight"], d["a"], d["b"], g, low.cuda(), scale=d["scale"])[0]
    # the same sums with every x (dy) of 2^-133, and the narrow product off by as much once more
    f = {name: t.double().abs() if t.is_floating_point() else t.long() for name, t in c.items()}
    step, s = 2.0 ** -133, f["scale"][f["ids"]][:, None]
    a, b = f["a"][f["ids"]], f["b"][f["ids"]]                # [n, r, K], [n, N, r]
    ones = torch.ones(n, r, 1, dtype=torch.float64)
    slack_low = step * a.sum(2)
    slack_y = step * f["weight"].sum(1)[None] + s * torch.bmm(b, slack_low[:, :, None] + step * ones)[:, :, 0]
    slack_dx = step * f["weight"].sum(0)[None] + s * torch.bmm(a.transpose(1, 2).contiguous(),
                                                               step * b.sum(1)[:, :, None] + step * ones)[:, :, 0]
    for got, want, size, terms, slack in ((kept, *(t[1] for t in (ref.forward(c), ref.forward(c, True))), k, slack_low),
                                          (y, *(t[0] for t in (ref.forward(c), ref.forward(c, True))), k + r, slack_y),
                                          (dx, *(t[0] for t in (ref.backward(c, low), ref.backward(c, low, True))), n_out + r, slack_dx)):
        err = (got.cpu().double() - want).abs()
        assert (err <= ref.bound(want, size, terms, torch.float32) + slack).all()
