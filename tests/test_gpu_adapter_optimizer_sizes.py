"""The adapters' optimizer over more parameters than one launch may have threads.  Needs an MI355X."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_target", [False, True])
def test_more_than_two_to_the_thirty_second_parameters(with_target):
    """2047 adapters of rank 81 beside a layer of 13440 x 512 have 4.6e9 parameters.  Elements at the ends of every launch and
    on both sides of 2^31 and 2^32 take Adam's step, what has no gradient stays."""
    from flatland_marl_amd.adapters import AdapterAdam
    n = 2047 * 81 * (13440 + 512) * 2
    assert n > 2 ** 32
    if torch.cuda.mem_get_info()[0] < (5 * 4 + 2) * n:
        pytest.skip("%d GB of device memory needed" % ((5 * 4 + 2) * n >> 30))
    flat = torch.zeros(n, device="cuda")
    opt = AdapterAdam(types.SimpleNamespace(flat=flat), lr=0.5)
    target = types.SimpleNamespace(flat=torch.zeros(n, device="cuda")) if with_target else None
    places = sorted({p + d for p in (0, 2 ** 30, 2 ** 31, 3 * 2 ** 30, 2 ** 32, n) for d in (-2, -1, 0, 1) if 0 <= p + d < n})
    at = torch.tensor(places, device="cuda")
    opt.grads[at] = 3.0
    opt.step(target, 0.25 if with_target else None)
    # the first step: -lr * g / (|g| + eps)
    assert torch.allclose(flat[at], torch.full((len(places),), -0.5, device="cuda"), rtol=1e-6)
    if with_target:
        assert torch.allclose(target.flat[at], torch.full((len(places),), -0.125, device="cuda"), rtol=1e-6)
    moved = sum(int(torch.count_nonzero(part)) for part in flat.split(1 << 30))
    assert moved == len(places)
    del flat, opt, target
    torch.cuda.empty_cache()
