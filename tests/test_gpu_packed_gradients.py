"""Clipping of the network's gradient in the packed form (flm_dqn_grad_clip), piece by piece against 64-bit forms.  Needs an
MI355X."""
import math

import pytest
import torch

from tests.test_gpu_adapter_training import _agent, _batch

pytestmark = pytest.mark.gpu


def _pieces(Rp, T1, n, rails4):
    """(first, end) of what the packed form holds: the convolution with the advantage stream's packed weights, its biases with
    the value stream's packed weights, the value stream's biases with the output layers."""
    a1_w, block, used = 64 * T1 + 64, 512 * 64 * 3 * Rp, 512 * 64 * 3 * rails4
    a1_b = a1_w + block
    v1_w = a1_b + 512
    return [(0, a1_w + used), (a1_b, v1_w + used), (v1_w + block, n)]


def _clipped(g, factor):
    """What a clipped element may be: the 64-bit product rounded once to fp32."""
    want = g.double() * factor
    return want, 2.0 ** -24 * want.abs() * (1 + 2.0 ** -20) + 2.0 ** -149


@pytest.mark.parametrize("inf_norm", [0, 1])
@pytest.mark.parametrize("limit", [0.3, 3.0])
@pytest.mark.parametrize("Rp,rails4", [(9, 4), (5, 4), (8, 8), (12, 12), (4, 4)])
def test_every_piece_is_counted_and_scaled(Rp, rails4, limit, inf_norm):
    """rails4 == Rp: there are no empty rows, and nothing but the pieces counts, whatever rcb holds."""
    from flatland_marl_amd import _lib
    T1, NA = 13, 2
    n = _lib.query("flm_dqn_param_count", 3 * Rp, T1, NA)
    gen = torch.Generator().manual_seed(Rp * 16 + rails4)
    g = torch.randn(n, generator=gen)
    pieces = _pieces(Rp, T1, n, rails4)
    (_, _), (a1_b, _), (v1_b, _) = pieces
    keep = torch.zeros(n, dtype=torch.bool)
    for lo, hi in pieces:
        keep[lo:hi] = True
    rcb = torch.rand(64, generator=gen) * 5                  # (large: a product that should not count would show)
    bias = torch.cat([g[a1_b:a1_b + 512], g[v1_b:v1_b + 512]]).double()
    empty = (bias[:, None] * rcb.double()).flatten().repeat(3 * (Rp - rails4))
    every = torch.cat([g[keep].double(), empty])
    norm = every.abs().max().item() if inf_norm else math.sqrt(math.fsum((every * every).tolist()))
    limit *= norm
    buf = torch.where(keep, g, torch.tensor(float("nan"))).cuda()
    r = rcb.cuda()
    work = torch.empty(_lib.GRAD_WORKSPACE, dtype=torch.float64, device="cuda")
    out = torch.full((), -1.0, device="cuda")
    _lib.launch(buf.device, "flm_dqn_grad_clip", buf.data_ptr(), Rp, T1, NA, rails4, 1, r.data_ptr(), limit, inf_norm, work.data_ptr(),
                out.data_ptr())
    assert abs(out.item() - norm) <= 2.0 ** -23 * norm
    got = buf.cpu()
    assert torch.isnan(got[~keep]).all()                     # what lies between the pieces is not touched
    want, tol = _clipped(g, min(1.0, limit / (norm + 1e-6)))
    # (the factor's 64-bit norm may differ in its last bits: far below half a step of fp32)
    assert ((got.double() - want).abs() <= tol)[keep].all()
    assert torch.equal(r.cpu(), rcb)


@pytest.mark.parametrize("inf_norm", [0, 1])
def test_an_infinite_norm_without_empty_rows(inf_norm):
    """An infinite bias gradient and no empty rows: the finite elements become zero, none of them NaN."""
    from flatland_marl_amd import _lib
    Rp, T1, NA = 4, 13, 2
    n = _lib.query("flm_dqn_param_count", 3 * Rp, T1, NA)
    g = torch.ones(n)
    a1_b = _pieces(Rp, T1, n, Rp)[1][0]
    g[a1_b + 3] = float("inf")
    buf, r = g.cuda(), torch.zeros(64).cuda()
    work = torch.empty(_lib.GRAD_WORKSPACE, dtype=torch.float64, device="cuda")
    out = torch.empty((), device="cuda")
    _lib.launch(buf.device, "flm_dqn_grad_clip", buf.data_ptr(), Rp, T1, NA, Rp, 1, r.data_ptr(), 1.0, inf_norm, work.data_ptr(),
                out.data_ptr())
    assert math.isinf(out.item())
    got = buf.cpu()
    assert torch.isnan(got[a1_b + 3]) and int(torch.isnan(got).sum()) == 1 and got.nan_to_num().abs().max() == 0


def test_a_learn_step_clips_every_piece():
    """The gradient that DQNAgent.learn_obs leaves in the packed form, clipped, against the same step's without a bound."""
    from flatland_marl_amd import _lib
    Rp, T1, B, rails, ps, NA = 24, 33, 64, 6, 800, 2
    dev, _ = _batch(B, Rp, T1, ps, rails, 3)
    agents = []
    for limit in (1e30, None):
        agent = _agent(Rp, T1, limit if limit is not None else 0.4 * agents[0].last_grad_norm.item())
        agent.optimizer._ensure()
        agent.optimizer.grads.fill_(-7.0)
        agent.learn_obs(dev, 0.99, ps, rails_used=rails)
        assert agent.optimizer._compact is not None
        agents.append(agent)
    free, bound = agents
    rails4 = free.optimizer._compact[3]
    n = free.optimizer.grads.numel()
    assert n == _lib.query("flm_dqn_param_count", 3 * Rp, T1, NA)
    g, got = free.optimizer.grads.cpu(), bound.optimizer.grads.cpu()
    norm = free.last_grad_norm.item()
    assert bound.last_grad_norm.item() == norm
    keep = torch.zeros(n, dtype=torch.bool)
    for lo, hi in _pieces(Rp, T1, n, rails4):
        keep[lo:hi] = True
        assert (g[lo:hi] != 0).any()
    assert (g[~keep] == -7.0).all() and (got[~keep] == -7.0).all()
    # (the norm is known here as its fp32 rounding: half a step of the factor)
    want, tol = _clipped(g, min(1.0, bound.max_grad_norm / (norm + 1e-6)))
    assert ((got.double() - want).abs() <= tol + 2.0 ** -23 * want.abs())[keep].all()


def test_a_bad_bound_is_the_same_error_in_either_form():
    agent = _agent(8, 17)
    for rails in (None, (8, 17, 2, 4, torch.zeros(64).cuda(), True)):
        for bad in (-1.0, float("nan")):
            with pytest.raises(ValueError):
                agent.optimizer.clip_grad_norm_(bad, rails=rails)
