"""Groups of replayed transitions.  Needs an MI355X."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _add(mem, first, n, groups=True):
    """n transitions whose states, actions and groups all tell which they are."""
    which = torch.arange(first, first + n)
    rows = (which % 251).to(torch.uint8)[:, None].expand(n, 16).contiguous().cuda()
    mem.add(rows, which.cuda(), which.float().cuda(), rows, torch.zeros(n).cuda(), groups=which.to(torch.int32).cuda() if groups else None)


def test_groups_are_those_of_the_drawn_transitions():
    from flatland_marl_amd.replay import DeviceReplay
    mem = DeviceReplay(40, 16, "cuda", seed=5)
    mem.keep_groups()
    _add(mem, 0, 40)
    for turn in range(3):
        s, a, *_ = mem.sample(16)
        drawn = a.clone()
        _add(mem, 40 + 40 * turn, 40)                        # every place of the ring is taken anew before the groups are read
        assert torch.equal(mem.sampled_groups(), drawn.int())
        first = mem.sampled_groups()
        mem.sample(16)
        assert torch.equal(first, drawn.int())               # (a tensor of the caller's)


def test_transitions_drawn_before_groups_were_kept():
    from flatland_marl_amd.replay import DeviceReplay
    mem = DeviceReplay(20, 16, "cuda", seed=5)
    _add(mem, 0, 20, groups=False)
    mem.sample(8)
    mem.keep_groups()
    _add(mem, 20, 20)
    assert mem.sampled_groups().tolist() == [-1] * 8
    mem.sample(8)
    assert (mem.sampled_groups() >= 20).all()
