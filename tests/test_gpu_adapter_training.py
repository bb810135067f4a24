"""The DQN with a bounded gradient norm and with low-rank adapters per map: the agent's, the policy's and the trainer's paths
through the adapter and clipping calls, against plain 64-bit PyTorch.  Needs an MI355X."""
import math
import types

import numpy as np
import pytest
import torch

from tests.test_gpu_train import _setup
from tests.torch_ref_dqn import TorchDuelingDQN

pytestmark = pytest.mark.gpu


def _agent(Rp, T1, max_grad_norm=None, seed=0, tau=1e-3, cls=None, double_dqn=True, lr=1e-3, NA=2):
    from flatland_marl_amd.agent import DQNAgent
    args = types.SimpleNamespace(prediction_depth=T1 - 1, lr=lr, buffer_size=64, batch_size=32, update_every=10, gamma=0.99, tau=tau)
    if max_grad_norm is not None:
        args.max_grad_norm = max_grad_norm
    torch.manual_seed(seed)
    agent = (cls or DQNAgent)(args, action_space=NA, bitmap_height=3 * Rp, double_dqn=double_dqn)
    with torch.no_grad():                                    # a target network of its own
        agent.qnetwork_target.flat_params().add_(0.02 * torch.randn_like(agent.qnetwork_target.flat_params()))
    return agent


def _batch(B, Rp, T1, ps, rails, seed, NA=2):
    """uint8 observations with `rails` used rails, and the rest of the experiences."""
    rng = np.random.default_rng(seed)

    def obs():
        o = np.zeros((B, 3, ps), np.uint8)
        planes = np.zeros((B, 3, Rp, T1), np.int64)
        planes[:, 0, :rails] = rng.integers(-1, 2, (B, rails, T1)) * (rng.random((B, rails, T1)) < 0.2)
        planes[:, 1:, :rails] = rng.integers(0, 4, (B, 2, rails, T1)) * (rng.random((B, 2, rails, T1)) < 0.3)
        o[:, :, :Rp * T1] = planes.reshape(B, 3, -1).astype(np.int8).view(np.uint8)
        return torch.from_numpy(o), torch.from_numpy(planes.reshape(B, 1, 3 * Rp, T1)).double()

    (s, sf), (n, nf) = obs(), obs()
    a = torch.from_numpy(rng.integers(0, NA, B))
    r, d = torch.from_numpy(rng.normal(size=B).astype(np.float32)), torch.from_numpy((rng.random(B) < 0.3).astype(np.float32))
    dev = tuple(t.cuda() for t in (s, a, r, n, d))
    return dev, (sf, a, r.double(), nf, d.double())


def test_learn_clips_the_gradient():
    Rp, T1, B = 8, 17, 24
    _, (s, a, r, n, d) = _batch(B, Rp, T1, 144, Rp, 1)
    batch = tuple(t.float().cuda() if t.dtype == torch.float64 else t.cuda() for t in (s, a, r, n, d))
    free = _agent(Rp, T1)
    free.learn(batch, 0.99)
    g = free.optimizer.grads.double()
    norm = math.sqrt(float(g.square().sum()))
    assert free.last_grad_norm is None
    for limit in (0.3 * norm, 3 * norm):
        agent = _agent(Rp, T1, limit)
        agent.learn(batch, 0.99)
        assert abs(agent.last_grad_norm.item() - norm) <= 2.0 ** -23 * norm
        want = g * min(1.0, limit / (norm + 1e-6))
        got = agent.optimizer.grads.double()
        assert ((got - want).abs() <= 2.0 ** -22 * want.abs()).all()
        assert torch.equal(agent.optimizer.m, (agent.optimizer.grads * np.float32(1 - 0.9)))
    assert torch.equal(agent.qnetwork_local.flat_params(), free.qnetwork_local.flat_params())     # the loose limit changed nothing


def test_clipping_in_the_packed_form_is_the_same():
    """Over the used rails, the two weight blocks packed and the gradient under the empty rows left to the optimizer pass:
    the norm counts all of it, and the steps are those of the whole gradient."""
    from flatland_marl_amd.agent import DQNAgent

    class Whole(DQNAgent):                                   # (a soft_update of its own: the whole gradient is written)
        def soft_update(self, *args):
            super().soft_update(*args)

    Rp, T1, B, rails, ps, lr = 24, 33, 64, 6, 800, 1e-3
    first = _agent(Rp, T1, 1e30, lr=lr)
    dev, _ = _batch(B, Rp, T1, ps, rails, 3)
    first.learn_obs(dev, 0.99, ps, rails_used=rails)
    limit = 0.4 * first.last_grad_norm.item()
    packed, whole = _agent(Rp, T1, limit, lr=lr), _agent(Rp, T1, limit, lr=lr, cls=Whole)
    for step in range(3):
        dev, _ = _batch(B, Rp, T1, ps, rails, 3 + step)
        packed.learn_obs(dev, 0.99, ps, rails_used=rails)
        whole.learn_obs(dev, 0.99, ps, rails_used=rails)
        norm, clipped = whole.last_grad_norm.item(), whole.optimizer.grads.double()
        # (the gradient under the empty rows: products rounded to fp32 here, none there; the networks differ by rounding
        # from the second step on)
        assert abs(packed.last_grad_norm.item() - norm) <= (2.0 ** -22 if step == 0 else 2.0 ** -16) * norm
        assert abs(math.sqrt(float(clipped.square().sum())) - min(limit, norm)) <= 1e-5 * limit
    assert packed.optimizer._compact is not None             # it did run in the packed form
    a, b = packed.qnetwork_local.flat_params(), whole.qnetwork_local.flat_params()
    # Adam's quotient m / (sqrt(v) + eps) moves with the gradient's relative error; where a gradient nearly vanishes
    # against what rounding leaves of it, a step of lr may turn: not more than a few such weights
    far = (a - b).abs() > 3 * lr * 2.0 ** -10 + 2.0 ** -22 * b.abs()
    assert far.float().mean().item() < 1e-3
    # a subset of rails the optimizer does not know as equal: the whole gradient is used instead of refusing
    again = _agent(Rp, T1, limit)
    again.optimizer.m
    again.learn_obs(dev, 0.99, ps, rails_used=rails)
    assert again.last_grad_norm.item() > 0


def _reference(agent, network, adapters, ids, x, absolute=False):
    """q, hidden activations and features in 64 bits; absolute: of absolute values throughout (error bounds)."""
    f = (lambda t: t.detach().cpu().double().abs()) if absolute else (lambda t: t.detach().cpu().double())
    sd = {k: f(v) for k, v in network.state_dict().items()}
    x = x.abs() if absolute else x
    feat = torch.relu(torch.einsum("bht,ct->bch", x[:, 0], sd["conv1.weight"][:, 0, 0]) + sd["conv1.bias"][None, :, None]).flatten(1)
    pre = {}
    for part in ("adv", "val"):
        y = feat @ sd["fc1_%s.weight" % part].t() + sd["fc1_%s.bias" % part]
        a, b = f(getattr(adapters, "a_" + part)), f(getattr(adapters, "b_" + part))
        for e in range(adapters.n_adapters):
            rows = (ids == e).nonzero().flatten()
            if len(rows):
                y[rows] += adapters.scale * ((feat[rows] @ a[e].t()) @ b[e].t())
        pre[part] = y
    ha, hv = torch.relu(pre["adv"]), torch.relu(pre["val"])
    adv, val = ha @ sd["fc2_adv.weight"].t() + sd["fc2_adv.bias"], hv @ sd["fc2_val.weight"].t() + sd["fc2_val.bias"]
    q = val + adv + adv.mean(1, keepdim=True) if absolute else val + adv - adv.mean(1, keepdim=True)
    return q, (ha, hv), feat


def _with_adapters(agent, E, r, seed=5):
    ad = agent.attach_adapters(E, r, alpha=2.0 * r)
    g = torch.Generator().manual_seed(seed)
    for bank, size in ((ad, 0.05), (agent.adapters_target, 0.04)):
        for name in ("b_adv", "b_val"):
            t = getattr(bank, name)
            t.copy_(size * torch.randn(t.shape, generator=g))
    return ad


@pytest.mark.parametrize("B,E,r", [(1, 2, 4), (9, 3, 5), (70, 4, 16)])
def test_adapted_q_values_against_64_bits(B, E, r):
    from flatland_marl_amd.adapters import group_rows
    Rp, T1, ps = 8, 17, 144
    agent = _agent(Rp, T1)
    ad = agent.attach_adapters(E, r, alpha=2.0 * r)
    dev, (x, *_) = _batch(B, Rp, T1, ps, 6, B)
    ids = torch.from_numpy(np.random.default_rng(B).integers(-1, E, B))
    groups = group_rows(ids.cuda(), E)
    plain = agent.qnetwork_local.forward_obs(dev[0], ps)
    fresh = ad.q_values(agent.qnetwork_local, dev[0], ps, groups)
    # one rounding a matrix instruction (T1, 64 * 3 * Rp and 512 terms; six instructions per 16) and 64 for each layer's rest
    c = (6 * (T1 + 192 * Rp + 512) / 16 + 3 * 64) * 2.0 ** -24
    size = _reference(agent, agent.qnetwork_local, ad, ids, x, True)[0]
    assert ((fresh - plain).cpu().double().abs() <= 2 * c * size).all()          # new adapters change nothing
    _with_adapters(agent, E, r)
    ad = agent.adapters
    got = ad.q_values(agent.qnetwork_local, dev[0], ps, groups)
    want, size = _reference(agent, agent.qnetwork_local, ad, ids, x)[0], _reference(agent, agent.qnetwork_local, ad, ids, x, True)[0]
    assert ((got.cpu().double() - want).abs() <= c * size).all()
    assert (got[ids.cuda() < 0] - plain[ids.cuda() < 0]).abs().max().item() <= 2 * c * size.max().item() if (ids < 0).any() else True
    empty = ad.q_values(agent.qnetwork_local, dev[0][:0], ps, group_rows(ids[:0].cuda(), E))
    assert empty.shape == (0, 2)


@pytest.mark.parametrize("double_dqn", [True, False])
@pytest.mark.parametrize("B,E,r,limit", [(24, 3, 4, None), (70, 5, 16, 0.05)])
def test_adapter_learn_step_against_64_bits(B, E, r, limit, double_dqn):
    Rp, T1, ps, gamma = 8, 17, 144, 0.9
    agent = _agent(Rp, T1, limit, tau=0.25, double_dqn=double_dqn)
    ad = _with_adapters(agent, E, r)
    dev, (s, a, rew, sn, done) = _batch(B, Rp, T1, ps, 6, 10 + B)
    ids = torch.from_numpy(np.random.default_rng(B).integers(-1, E, B))
    ids[ids == 1] = 0                                        # adapter 1 has no rows
    nets = [agent.qnetwork_local.flat_params().clone(), agent.qnetwork_target.flat_params().clone()]
    old, old_t = ad.flat.clone(), agent.adapters_target.flat.clone()
    start = {k: v.cpu().double() for k, v in ad.state_dict().items()}
    args = (agent, agent.qnetwork_local, ad, ids)
    q, (ha, hv), feat = _reference(*args, s)
    qa, _, feat_a = _reference(*args, s, True)
    qn = _reference(*args, sn)[0]
    target_args = (agent, agent.qnetwork_target, agent.adapters_target, ids, sn)
    qt, qta = _reference(*target_args)[0], _reference(*target_args, True)[0]
    rows = torch.arange(B)
    if double_dqn:
        y = rew + gamma * qt[rows, qn.argmax(1)] * (1 - done)
        loss, dq_taken = ((q[rows, a] - y) ** 2).mean(), 2 * (q[rows, a] - y) / B
    else:                                                    # the reference's [B, B] broadcast
        y = rew[None] + gamma * qt.max(1).values[:, None] * (1 - done)[None]
        loss, dq_taken = ((q[rows, a][None] - y) ** 2).mean(), 2 * (q[rows, a][None] - y).mean(0) / B
    c = (6 * (T1 + 192 * Rp + 512) / 16 + 3 * 64) * 2.0 ** -24
    dq_error = 2 * c * (qa[rows, a] + gamma * qta.max()) / B  # what the Q-values' rounding makes of dq

    def backward(dq_row, absolute):
        f = (lambda t: t.abs()) if absolute else (lambda t: t)
        sd = {k: f(v.detach().cpu().double()) for k, v in agent.qnetwork_local.state_dict().items()}
        dq = torch.zeros(B, 2, dtype=torch.float64)
        dq[rows, a] = dq_row
        mean = dq.mean(1, keepdim=True)
        dadv = dq + mean if absolute else dq - mean
        out = {}
        for part, dh in (("adv", (dadv @ sd["fc2_adv.weight"]) * (ha > 0)), ("val", (dq.sum(1, keepdim=True) @ sd["fc2_val.weight"]) * (hv > 0))):
            ga, gb = torch.zeros_like(start["a_" + part]), torch.zeros_like(start["b_" + part])
            for e in range(E):
                pick = (ids == e).nonzero().flatten()
                if len(pick):
                    x = feat_a[pick] if absolute else feat[pick]
                    u = ad.scale * (dh[pick] @ f(start["b_" + part][e]))
                    ga[e] = u.t() @ x
                    gb[e] = ad.scale * (dh[pick].t() @ (x @ f(start["a_" + part][e]).t()))
            out["a_" + part], out["b_" + part] = ga, gb
        return out

    agent.learn_adapters(dev, ids.cuda(), gamma, ps)
    want, size, extra = backward(dq_taken, False), backward(dq_taken.abs(), True), backward(dq_error, True)
    got = {k: v.cpu().double() for k, v in ad.views(agent.adapter_optimizer.grads).items()}
    factor = 1.0
    if limit is not None:
        norm = math.sqrt(sum(float(v.square().sum()) for v in want.values()))
        factor = min(1.0, limit / (norm + 1e-6))
        assert factor < 1.0
        slack = math.sqrt(sum(float((c * size[k] + extra[k]).square().sum()) for k in want))
        assert abs(agent.last_grad_norm.item() - norm) <= slack + 2.0 ** -23 * norm
    for k in want:
        slack = factor * (2 * c * size[k] + extra[k]) + (abs(want[k]) * 1e-4 if limit is not None else 0) + 1e-12
        assert ((got[k] - factor * want[k]).abs() <= slack).all(), k
        assert (got[k][1] == 0).all()
    assert abs(agent.last_loss.item() - loss.item()) <= (2 * (q[rows, a].abs().max() + y.abs().max()) * c * 2 * (qa.max() + qta.max())).item() + 1e-6 * loss.item()
    # Adam's first step and the target's soft update; the networks stay as they are
    g = agent.adapter_optimizer.grads.double()
    new = old.double() - 1e-3 * g / (g.abs() + 1e-8)
    assert ((ad.flat.double() - new).abs() <= 2.0 ** -22 * new.abs() + 1e-3 * 2.0 ** -18).all()
    mixed = 0.25 * ad.flat.double() + 0.75 * old_t.double()
    assert ((agent.adapters_target.flat.double() - mixed).abs() <= 2.0 ** -22 * (ad.flat.abs() + old_t.abs()).double()).all()
    assert torch.equal(nets[0], agent.qnetwork_local.flat_params()) and torch.equal(nets[1], agent.qnetwork_target.flat_params())


def test_training_with_an_adapter_per_environment(tmp_path):
    ro, agent, _ = _setup(E=6)
    ad = agent.attach_adapters(3, 8, lr=1e-3)
    from flatland_marl_amd.train import BatchedTrainer
    of_env = [0, 1, 2, 0, -1, 1]
    tr = BatchedTrainer(ro, agent, start_eps=0.3, max_learns_per_step=2, max_steps=40, adapter_of_env=of_env)
    nets = agent.qnetwork_local.flat_params().clone()
    before = ad.flat.clone()
    # one step by hand: every stored transition carries its environment's adapter
    ro.reset()
    assert tr.step(train=True) > 0
    n = ro.E * ro.A
    slot, req = tr.replay._slot[:n].cpu(), tr.replay._req[:n].cpu()
    for k in range(int((slot >= 0).sum())):
        i = int((slot == k).nonzero()[0])
        assert int(tr.replay.group[k]) == of_env[int(req[i]) // ro.A]
    out = tr.run_episode(train=True)
    assert out["learns"] > 0 and torch.isfinite(agent.last_loss).all()
    used = len(tr.replay)
    assert set(tr.replay.group[:used].tolist()) == {-1, 0, 1, 2} and bool((tr.replay.group[used:-1] == -1).all())
    assert torch.equal(nets, agent.qnetwork_local.flat_params())
    assert torch.isfinite(ad.flat).all() and not torch.equal(before, ad.flat)
    # what an environment's agents are shown is the network with its adapter
    policy = tr.policy
    obs = torch.zeros((4, 3, ro.b.plane_stride), dtype=torch.uint8, device="cuda")
    obs[:, 1, :600] = 1
    agents = torch.tensor([0, ro.A, 4 * ro.A, 5 * ro.A + 3], dtype=torch.int32, device="cuda")
    q = policy._adapted_q_values(ro, obs, agents, None)
    plain = agent.qnetwork_local.forward_obs(obs, ro.b.plane_stride)
    assert torch.equal(q[1], q[3]) and not torch.equal(q[0], q[1]) and torch.allclose(q[2], plain[2], rtol=1e-4, atol=1e-5)
    policy.chunk_bytes = 8 * ad.inputs                       # two rows at a time
    assert torch.allclose(policy._adapted_q_values(ro, obs, agents, None), q, rtol=1e-5, atol=1e-6)
    # saved and loaded
    agent.save(str(tmp_path / "net"))
    kept = ad.flat.clone()
    ad.flat.zero_()
    agent.load(str(tmp_path / "net"))
    assert torch.equal(ad.flat, kept)


def test_refusals():
    from flatland_marl_amd.adapters import NetworkAdapters, group_rows
    from flatland_marl_amd.train import BatchedTrainer, DQNPolicy
    ro, agent, tr = _setup(E=2)
    dev, _ = _batch(4, 100, 151, ro.b.plane_stride, 5, 1)
    with pytest.raises(ValueError):
        agent.learn_adapters(dev, torch.zeros(4, dtype=torch.int32).cuda(), 0.9, ro.b.plane_stride)
    with pytest.raises(ValueError):
        DQNPolicy(agent, adapter_of_env=torch.zeros(2, dtype=torch.int32).cuda())
    for bad in ((0, 4), (2048, 4), (3, 0), (3, 129)):
        with pytest.raises(ValueError):
            NetworkAdapters(agent.qnetwork_local, *bad)
    ad = agent.attach_adapters(2, 4)
    for kw in (dict(adapter_of_env=[0]), dict(adapter_of_env=[0, 1], crash_penalty=True), dict(adapter_of_env=[0, 1], switch2switch=True)):
        with pytest.raises(ValueError):
            BatchedTrainer(ro, agent, **kw)
    with pytest.raises(ValueError):                          # a group for three rows, observations for four
        ad.q_values(agent.qnetwork_local, dev[0], ro.b.plane_stride, group_rows(torch.zeros(3, dtype=torch.int32).cuda(), 2))
    with pytest.raises(ValueError):
        ad.q_values(agent.qnetwork_local, dev[0].float(), ro.b.plane_stride, group_rows(torch.zeros(4, dtype=torch.int32).cuda(), 2))
    ids = torch.zeros(4, dtype=torch.int32).cuda()
    groups = group_rows(ids, 2)
    net, stride = agent.qnetwork_local, ro.b.plane_stride
    with pytest.raises(ValueError):                          # observations, results and features that are not where they should be
        ad.q_values(net, dev[0].cpu(), stride, groups)
    for kw in (dict(out=torch.zeros(3, 2).cuda()), dict(out=torch.zeros(4, 2)), dict(out=torch.zeros(4, 2).cuda().half()),
               dict(features=torch.zeros(4 * ad.inputs - 1).cuda()), dict(features=torch.zeros(4 * ad.inputs))):
        with pytest.raises(ValueError):
            ad.q_values(net, dev[0], stride, groups, **kw)
    for i in (1, 2, 4):                                      # an action, a reward, a flag too few
        short = list(dev)
        short[i] = short[i][:3]
        with pytest.raises(ValueError):
            agent.learn_adapters(short, ids, 0.9, stride)
    policy = DQNPolicy(agent, adapter_of_env=torch.zeros(1, dtype=torch.int32).cuda())
    with pytest.raises(ValueError):
        policy._adapted_q_values(ro, dev[0], ids, None)
    for groups_of in (None, ids[:3]):                        # groups without keep_groups(), too few of them
        if groups_of is not None:
            tr.replay.keep_groups()
        with pytest.raises(ValueError):
            tr.replay.add(dev[0], dev[1], dev[2], dev[3], dev[4], groups=ids if groups_of is None else groups_of)
        with pytest.raises(ValueError):
            tr.replay.sampled_groups()
    before = ad.state_dict()
    bad = dict(before, b_val=before["b_val"][:1])
    bad["a_adv"] = before["a_adv"] + 1
    with pytest.raises(ValueError):
        ad.load_state_dict(bad)
    assert all(torch.equal(before[k], v) for k, v in ad.state_dict().items())
    with pytest.raises(ValueError):
        agent.optimizer.clip_grad_norm_(1.0, rails=(100, 151, 2, 8, None, False))
