"""Global gradient norm and clipping against plain 64-bit sums.  Needs an MI355X."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SETS = [[1], [7], [64], [0, 3, 0], [1, 2, 3, 4, 5, 6, 7, 8, 9], [65536], [65537], [5, 70000, 8191, 8192, 8193, 1],
        [100] * 111, [100] * 112, [100] * 113, [37, 4099] * 200, [3000001, 12], [20000000], [40000003, 5, 40000000]]


def _grads(sizes, kind, seed=0, scale=0.1):
    g = torch.Generator().manual_seed(seed)
    kinds = TYPES if kind is None else [kind]
    return [(torch.randn(n, generator=g) * scale).to(kinds[i % len(kinds)]) for i, n in enumerate(sizes)]


def _norm(grads):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def _close(got, want, kind):
    # one rounding of a 64-bit product to fp32, one to the type
    step = torch.finfo(kind).eps / 2 + 2.0 ** -24
    tiny = torch.finfo(kind).smallest_normal * torch.finfo(kind).eps
    assert ((got.double() - want).abs() <= step * want.abs() * (1 + step) + tiny).all()


@pytest.mark.parametrize("kind", TYPES + [None], ids=str)
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: "%dx%d" % (len(s), sum(s)))
def test_norm_and_clip(sizes, kind):
    from flatland_marl_amd.gradients import clip_grad_norm_, grad_norm
    host = _grads(sizes, kind)
    dev = [g.cuda() for g in host]
    want = _norm(host)
    assert abs(grad_norm(dev).item() - want) <= 2.0 ** -23 * want       # (a 64-bit sum, rounded to fp32)
    for limit in (0.5 * want, 2 * want + 1):
        outs = [torch.full_like(g, float("nan")) for g in dev]
        before = [g.clone() for g in dev]
        norm = clip_grad_norm_(dev, limit, out=outs)
        assert abs(norm.item() - want) <= 2.0 ** -23 * want
        assert all(torch.equal(a, b) for a, b in zip(before, dev))
        factor = min(1.0, limit / (want + 1e-6))
        for g, o in zip(host, outs):
            _close(o.cpu(), g.double() * factor, g.dtype)
        inplace = [g.clone() for g in dev]
        norm2 = clip_grad_norm_(inplace, limit)
        assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(inplace, outs))
        if factor == 1.0:
            assert all(torch.equal(a, b) for a, b in zip(inplace, dev))
    top = max([float(g.abs().max()) for g in host if g.numel()], default=0.0)
    assert grad_norm(dev, norm_type=float("inf")).item() == top


def test_pieces_of_one_buffer_at_odd_places():
    from flatland_marl_amd.gradients import clip_grad_norm_
    for kind in TYPES:
        flat = (torch.randn(200001, generator=torch.Generator().manual_seed(2)) * 0.1).to(kind).cuda()
        keep = flat.clone()
        pieces = [flat[1:4], flat[5:70001], flat[70003:70004], flat[90000:200000]]
        want = _norm([p.cpu() for p in pieces])
        norm = clip_grad_norm_(pieces, 1.0)
        assert abs(norm.item() - want) <= 2.0 ** -23 * want
        mask = torch.zeros_like(flat, dtype=torch.bool)
        for lo, hi in ((1, 4), (5, 70001), (70003, 70004), (90000, 200000)):
            mask[lo:hi] = True
        assert torch.equal(flat[~mask], keep[~mask])
        _close(flat[mask].cpu(), keep[mask].cpu().double() * (1.0 / (want + 1e-6)), kind)


@pytest.mark.parametrize("scale", [1e-30, 1e30])
@pytest.mark.parametrize("sizes", [[1000], [300000]])
def test_squares_that_fp32_cannot_hold(sizes, scale):
    from flatland_marl_amd.gradients import clip_grad_norm_
    host = _grads(sizes, torch.float32, scale=scale)
    dev = [g.cuda() for g in host]
    want = _norm(host)
    norm = clip_grad_norm_(dev, 1.0)
    assert abs(norm.item() - want) <= 2.0 ** -23 * want
    for g, o in zip(host, dev):
        _close(o.cpu(), g.double() * min(1.0, 1.0 / (want + 1e-6)), torch.float32)


@pytest.mark.parametrize("n", [50, 400000])
def test_infinities_and_nan(n):
    from flatland_marl_amd.gradients import clip_grad_norm_, grad_norm
    for bad in (float("inf"), float("nan")):
        for kind in (2.0, float("inf")):
            g = _grads([n, 9], torch.float32)
            g[0][n // 2] = bad
            d = [t.cuda() for t in g]
            norm = grad_norm(d, norm_type=kind).item()
            assert math.isinf(norm) if math.isinf(bad) else math.isnan(norm)
            clip_grad_norm_(d, 1.0, norm_type=kind)
            if math.isnan(bad):
                assert all(torch.isnan(t).all() for t in d)
            else:                                                     # inf * 0 is NaN, the others become 0
                assert torch.isnan(d[0][n // 2]) and d[0].nan_to_num().abs().max() == 0 and (d[1] == 0).all()


def test_lists_with_none_shapes_and_zero_norm():
    from flatland_marl_amd.gradients import clip_grad_norm_, grad_norm
    w = torch.randn(40, 30).cuda().t()                                # dense, not contiguous
    ref = w.clone()
    want = _norm([w.cpu(), torch.ones(5)])
    norm = clip_grad_norm_([None, w, torch.ones(5).cuda(), torch.zeros(0).cuda()], 1.0)
    assert abs(norm.item() - want) <= 2.0 ** -23 * want
    _close(w.cpu(), ref.cpu().double() / (want + 1e-6), torch.float32)
    z = torch.zeros(100).cuda()
    assert clip_grad_norm_([z], 0.0).item() == 0 and (z == 0).all()
    assert grad_norm([torch.zeros(0).cuda()]).item() == 0 and grad_norm([]).item() == 0 and clip_grad_norm_([None], 1.0).item() == 0


def test_captured_and_replayed():
    from flatland_marl_amd.gradients import clip_grad_norm_
    for sizes in ([300, 17], [500000, 3, 90001]):
        grads = [g.cuda() for g in _grads(sizes, None)]
        outs = [torch.empty_like(g) for g in grads]
        clip_grad_norm_(grads, 1.0, out=outs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = clip_grad_norm_(grads, 1.0, out=outs)
        for turn in range(4):
            for g, new in zip(grads, _grads(sizes, None, seed=turn + 5, scale=0.2)):
                g.copy_(new)
            graph.replay()
            eager = [torch.empty_like(g) for g in grads]
            n2 = clip_grad_norm_(grads, 1.0, out=eager)
            torch.cuda.synchronize()
            assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(outs, eager)), turn


def test_shared_memory_is_refused():
    from flatland_marl_amd.gradients import clip_grad_norm_, grad_norm
    g, h = torch.ones(100).cuda(), torch.ones(100).cuda()
    for grads, out in (([g, g], None), ([g[:60], g[50:]], None), ([g, h], [h, g]), ([g, h], [torch.empty_like(g)] * 2)):
        with pytest.raises(ValueError):
            clip_grad_norm_(grads, 1.0, out=out)
    assert (g == 1).all() and abs(grad_norm([g, g]).item() - math.sqrt(200)) < 1e-5      # the norm alone may count twice
    for out in ([g], [g, h[:50]], [g, h.double()]):
        with pytest.raises(ValueError):
            clip_grad_norm_([g.clone(), h], 1.0, out=out)
