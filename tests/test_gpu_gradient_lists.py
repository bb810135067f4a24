"""Lists of gradients and outputs with holes.  Needs an MI355X."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_outputs_of_missing_gradients_are_left_alone():
    from flatland_marl_amd.gradients import clip_grad_norm_
    a, b = torch.full((300,), 3.0).cuda(), torch.full((50,), 4.0).cuda()
    want = [torch.empty_like(t) for t in (a, b)]
    norm = clip_grad_norm_([a, b], 1.0, out=want)
    spare = torch.full((300,), -1.0).cuda()
    for grads, place in (([None, a, b], (1, 2)), ([a, None, b], (0, 2)), ([a, b, None], (0, 1))):
        outs = [torch.full((300,), -1.0).cuda() if g is None else torch.empty_like(g) for g in grads]
        assert torch.equal(clip_grad_norm_(grads, 1.0, out=outs), norm)
        assert all(torch.equal(outs[i], w) for i, w in zip(place, want))
        assert all(torch.equal(o, spare) for g, o in zip(grads, outs) if g is None)
    with pytest.raises(ValueError):
        clip_grad_norm_([None, a], 1.0, out=[spare, None])
    assert (spare == -1.0).all()
