"""The agent's adapters over their whole life: saved and loaded, without rows, beside other buffers.  Needs an MI355X."""
import pytest
import torch

from tests.test_gpu_adapter_training import _agent, _batch, _with_adapters

pytestmark = pytest.mark.gpu
Rp, T1, PS, B, E, R = 8, 17, 144, 24, 3, 4


def _learn(agent, seed):
    dev, _ = _batch(B, Rp, T1, PS, 6, seed)
    ids = torch.randint(-1, E, (B,), generator=torch.Generator().manual_seed(seed)).cuda()
    agent.learn_adapters(dev, ids, 0.9, PS)


def test_training_goes_on_where_it_was_saved(tmp_path):
    """Values, target values, scale, moments and step count: two further steps give the same bits as without a break."""
    agent = _agent(Rp, T1)
    _with_adapters(agent, E, R)
    for seed in (1, 2):
        _learn(agent, seed)
    agent.save(str(tmp_path / "net"))
    other = _agent(Rp, T1, seed=9)
    other.attach_adapters(E, R, alpha=1.0)                    # (another scale)
    for seed in (5, 6, 7):                                   # moments and a step count of its own
        _learn(other, seed)
    other.load(str(tmp_path / "net"))
    assert other.adapters.scale == other.adapters_target.scale == agent.adapters.scale
    for seed in (3, 4):
        _learn(agent, seed)
        _learn(other, seed)
    for a, b in ((agent.adapters.flat, other.adapters.flat), (agent.adapters_target.flat, other.adapters_target.flat),
                 (agent.adapter_optimizer.m, other.adapter_optimizer.m), (agent.adapter_optimizer.v, other.adapter_optimizer.v)):
        assert torch.equal(a, b)
    assert agent.adapter_optimizer.step_count == other.adapter_optimizer.step_count == 4


def test_files_without_scale_and_optimizer(tmp_path):
    agent = _agent(Rp, T1)
    ad = _with_adapters(agent, E, R)
    name = str(tmp_path / "net")
    agent.save(name)
    torch.save({"local": ad.state_dict(), "target": agent.adapters_target.state_dict()}, name + ".adapters")
    kept, scale = ad.flat.clone(), ad.scale
    _learn(agent, 1)
    agent.load(name)
    assert torch.equal(ad.flat, kept) and ad.scale == scale and agent.adapter_optimizer.step_count == 0
    assert not agent.adapter_optimizer.m.any() and not agent.adapter_optimizer.v.any()


def test_a_refused_file_changes_nothing(tmp_path):
    agent = _agent(Rp, T1)
    _with_adapters(agent, E, R)
    name = str(tmp_path / "net")
    for change in ("rank", "target", "moments"):
        writer = _agent(Rp, T1, seed=4)
        _with_adapters(writer, E, R + 1 if change == "rank" else R)
        writer.save(name)
        state = torch.load(name + ".adapters", weights_only=True)
        if change == "target":
            state["target"]["b_val"] = state["target"]["b_val"][:1]
        elif change == "moments":
            state["optimizer"]["v"] = state["optimizer"]["v"][:-1]
        torch.save(state, name + ".adapters")
        before = [t.clone() for t in (agent.qnetwork_local.flat_params(), agent.qnetwork_target.flat_params(), agent.adapters.flat,
                                      agent.adapters_target.flat)]
        with pytest.raises(ValueError):
            agent.load(name)
        after = (agent.qnetwork_local.flat_params(), agent.qnetwork_target.flat_params(), agent.adapters.flat, agent.adapters_target.flat)
        assert all(torch.equal(a, b) for a, b in zip(before, after)), change


def test_what_stays_the_shared_networks():
    """act() and learn() with adapters attached: the network's values and training, the adapters untouched."""
    with_ad, without = _agent(Rp, T1), _agent(Rp, T1)
    _with_adapters(with_ad, E, R)
    dev, (s, a, r, n, d) = _batch(B, Rp, T1, PS, 6, 2)
    kept, kept_t = with_ad.adapters.flat.clone(), with_ad.adapters_target.flat.clone()
    state = s[0, 0].float().numpy()
    assert torch.equal(with_ad.act(state), without.act(state))
    batch = tuple(t.float().cuda() if t.is_floating_point() else t.cuda() for t in (s, a, r, n, d))
    for agent in (with_ad, without):
        agent.learn(batch, 0.9)
        agent.learn_obs(dev, 0.9, PS)
    assert torch.equal(with_ad.qnetwork_local.flat_params(), without.qnetwork_local.flat_params())
    assert torch.equal(with_ad.adapters.flat, kept) and torch.equal(with_ad.adapters_target.flat, kept_t)


def test_a_copy_has_the_same_scale_and_draws_nothing():
    from flatland_marl_amd.adapters import NetworkAdapters
    agent = _agent(Rp, T1)
    for rank, alpha in ((49, 1.0), (3, 1.3), (107, 0.7), (R, None)):
        torch.manual_seed(3)
        ad = NetworkAdapters(agent.qnetwork_local, 2, rank, alpha)
        state = torch.cuda.get_rng_state()
        other = ad.copy_for(agent.qnetwork_target)
        assert torch.equal(torch.cuda.get_rng_state(), state)
        assert other.scale == ad.scale and torch.equal(other.flat, ad.flat) and other.flat.data_ptr() != ad.flat.data_ptr()
        assert other.a_adv.data_ptr() == other.flat.data_ptr()


def test_no_observations_keep_what_their_gradients_take():
    from flatland_marl_amd.adapters import group_rows
    agent = _agent(Rp, T1)
    ad = _with_adapters(agent, E, R)
    dev, _ = _batch(4, Rp, T1, PS, 6, 1)
    q, kept = ad.q_values(agent.qnetwork_local, dev[0][:0], PS, group_rows(torch.zeros(0, dtype=torch.int32).cuda(), E), keep=True)
    assert q.shape == (0, 2)
    grads = torch.full_like(ad.flat, float("nan"))
    ad.gradients(kept, torch.empty((0, 2 * ad.outputs), device="cuda"), grads)
    assert (grads == 0).all()


def test_buffers_of_any_shape_receive_the_q_values():
    from flatland_marl_amd.adapters import group_rows
    agent = _agent(Rp, T1)
    ad = _with_adapters(agent, E, R)
    dev, _ = _batch(5, Rp, T1, PS, 6, 1)
    groups = group_rows(torch.tensor([0, 1, 2, -1, 0], dtype=torch.int32).cuda(), E)
    args = (agent.qnetwork_local, dev[0], PS, groups)
    want = ad.q_values(*args)
    for shape, rows in (((10,), (5 * ad.inputs + 3,)), ((7, 2), (5, ad.inputs)), ((2, 11), (9, ad.inputs)), ((3, 2, 2), (1, 5, ad.inputs))):
        out, features = torch.full(shape, -5.0).cuda(), torch.empty(rows).cuda()
        got = ad.q_values(*args, out=out, features=features)
        assert got.shape == (5, 2) and torch.equal(got, want) and got.data_ptr() == out.data_ptr()
        assert (out.view(-1)[10:] == -5.0).all()
