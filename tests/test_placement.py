"""Station placement (mobile_env.placement): the operators of mobile_env.learning together, as a
user runs them -- acting, advantages, loss and gradient, clipping, a step of the optimizer."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rollout(E=48, steps=23, cell=20):
    from mobile_env.placement import PlacementPolicy, collect, make_engine
    eng, count = make_engine(E, seed=7)
    torch.manual_seed(3)
    policy = PlacementPolicy(10, 100, hidden=16).to(eng.device)
    ro = collect(eng, policy, steps, cell, torch.Generator(device=eng.device).manual_seed(5))
    torch.cuda.synchronize()
    return eng, count, policy, ro


def _plain_loss(policy, ro, ref, gamma, lam, clip, kl, ent, value_coef):
    """The update's loss in float64 on the CPU, differentiated by autograd."""
    r, v = ro.reward.double(), ro.value.double()
    live = 1.0 - ro.done.double()
    nxt = torch.cat([v[1:], ro.last_value.double()[None]])
    delta = r + gamma * nxt - v
    adv = torch.zeros_like(r)
    run = torch.zeros_like(r[0])
    for t in range(len(r) - 1, -1, -1):
        run = delta[t] + gamma * lam * live[t] * run
        adv[t] = run
    ret = adv + v
    adv = (adv - adv.mean()) / (adv.std() + 1e-6)
    T, E, S = ro.action.shape
    w = ro.weight.double().expand(T, E, S)
    w = w / w.sum()
    logits, value = policy(ro.positions.double().flatten(0, 1))
    lp = torch.log_softmax(logits.view(T, E, S, -1), -1)
    L = lp.gather(-1, ro.action[..., None])[..., 0]
    ratio = (L - ro.logp.double()).exp()
    A = adv[..., None]
    l = -torch.minimum(ratio * A, ratio.clamp(1 - clip, 1 + clip) * A)
    d = ref.double() - L
    l = l + kl * (d.exp() - d - 1) + ent * (lp.exp() * lp).sum(-1)
    return (w * l).sum() + value_coef * (value.view(T, E) - ret).square().mean()


def test_rollout_places_stations_and_keeps_what_the_update_needs():
    eng, count, policy, ro = _rollout()
    assert ro.action.shape == (23, 48, 10) and ro.done.sum() == 48  # one episode end each
    xy = eng.bs_xy.long()
    a = ro.action[-1]
    want = torch.stack([a % 10, a // 10], -1) * 20 + 10
    assert torch.equal(xy, want)
    assert torch.equal(ro.weight.sum(1).int(), count)
    with torch.no_grad():
        logits, value = policy(ro.positions[4])
    L = torch.log_softmax(logits.double(), -1).gather(-1, ro.action[4][..., None])[..., 0]
    # (a product of 16 terms and its bias, then 100 exponentials and their sum, in float32)
    torch.testing.assert_close(ro.logp[4].double(), L, rtol=0, atol=128 * 2.0 ** -24 * 8)
    assert torch.equal(ro.value[4], value)
    eng.close()


def test_update_gradient_is_that_of_the_plain_loss():
    from mobile_env.learning import action_logp
    from mobile_env.placement import update
    eng, _, policy, ro = _rollout()
    with torch.no_grad():
        for p in policy.parameters():  # the policy has moved since it acted
            p.add_(0.05 * torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel()))
                   .to(p.device))
        logits, _ = policy(ro.positions.flatten(0, 1))
        ref, _ = action_logp(logits.view(*ro.action.shape, -1) * 0.9, ro.action)
    kw = dict(gamma=0.9, lam=0.95, clip=0.2, kl_coef=0.1, entropy_coef=0.01)
    twin = copy.deepcopy(policy).double().cpu()
    cpu = type(ro)(*(t.cpu() for t in ro))
    loss = _plain_loss(twin, cpu, ref.cpu(), 0.9, 0.95, 0.2, 0.1, 0.01, 0.5)
    loss.backward()
    total = torch.sqrt(sum((p.grad ** 2).sum() for p in twin.parameters()))
    opt = torch.optim.SGD(policy.parameters(), lr=1.0)
    before = [p.detach().clone() for p in policy.parameters()]
    out = update(policy, opt, ro, ref_logp=ref, max_grad_norm=float(total) / 2, **kw)
    got_loss = float(out["loss"]) + 0.5 * float(out["value_loss"])
    # float32 sums over 23 x 48 x 10 rows of order-one terms; a ratio within 2^-20 of a border may
    # take its other side (its row weighs 1 / 8,000)
    assert abs(got_loss - loss.item()) < 1e-4 * max(1.0, abs(loss.item()))
    assert abs(float(out["grad_norm"]) - float(total)) < 1e-3 * float(total)
    for p, b, q in zip(policy.parameters(), before, twin.parameters()):
        step = (b - p.detach()).double().cpu()          # lr 1: the clipped gradient
        want = q.grad / 2                               # the norm was twice what is allowed
        assert (step - want).norm() <= 2e-3 * want.norm() + 1e-6 * float(total), step.shape
    eng.close()


def test_training_runs():
    from mobile_env.placement import train_placement
    policy, rewards = train_placement(num_envs=64, cell=40, iterations=2, steps=20, epochs=2,
                                      seed=11)
    assert len(rewards) == 2 and all(-1.0 <= r <= 1.0 for r in rewards)
    assert all(torch.isfinite(p).all() for p in policy.parameters())


def test_stations_argument_is_checked():
    from mobile_env.placement import make_engine
    for bad in ((0, 3), (4, 2)):
        with pytest.raises(ValueError):
            make_engine(4, stations=bad)
    from mobile_env.placement import train_placement
    with pytest.raises(ValueError):
        train_placement(num_envs=4, cell=0)


def test_a_rollout_of_one_step_of_one_env():
    """One advantage has no deviation to be divided by."""
    from mobile_env.placement import train_placement
    policy, rewards = train_placement(num_envs=1, stations=(2, 2), cell=50, iterations=1, steps=1,
                                      epochs=1, seed=3)
    assert len(rewards) == 1
    assert all(torch.isfinite(p).all() for p in policy.parameters())
    with pytest.raises(ValueError):
        train_placement(num_envs=1, stations=(2, 2), cell=50, iterations=1, steps=0)


def test_actions_are_played_on_the_positions_they_were_chosen_for():
    """Over an episode's end, within a rollout and between two: what the policy saw is where the
    users stood when the step began, and the engine's rewards are those of its own lazy resets."""
    from mobile_env.placement import PlacementPolicy, collect, make_engine
    E, steps, cell = 24, 20, 20
    eng, _ = make_engine(E, seed=9)
    start = eng.obs[..., :2].clone()
    torch.manual_seed(4)
    policy = PlacementPolicy(10, 100, hidden=16).to(eng.device)
    g = torch.Generator(device=eng.device).manual_seed(6)
    # 7 steps first, so that the second rollout ends an episode in its midst; then whole episodes
    rollouts = [collect(eng, policy, n, cell, g) for n in (7, steps, 13, steps)]
    twin, _ = make_engine(E, seed=9)
    t = 0
    for k, ro in enumerate(rollouts):
        for i in range(len(ro.reward)):
            if t % 20 == 0:  # every episode starts from the same positions (the streams re-seed)
                assert torch.equal(ro.positions[i], start), (k, i)
            else:
                assert torch.equal(ro.positions[i], twin.obs[..., :2]), (k, i)
            a = ro.action[i]
            twin.set_bs_layout((torch.stack([a % 10, a // 10], -1) * cell + cell // 2).int())
            twin.step()
            assert torch.equal(ro.reward[i], twin.reward) and torch.equal(ro.done[i], twin.done)
            t += 1
        with torch.no_grad():
            last = policy(start if t % 20 == 0 else twin.obs[..., :2])[1]
        assert torch.equal(ro.last_value, last), k
    assert t == 60 and not torch.equal(start, twin.obs[..., :2])
    eng.close()
    twin.close()


def test_training_leaves_the_callers_generators_alone():
    from mobile_env.placement import PlacementPolicy, train_placement
    kw = dict(num_envs=8, stations=(2, 3), cell=50, iterations=1, steps=2, epochs=1, seed=3)
    for policy in (None, PlacementPolicy(3, 16)):
        cpu, gpu = torch.get_rng_state(), torch.cuda.get_rng_state()
        got, _ = train_placement(policy=policy, **kw)
        assert torch.equal(torch.get_rng_state(), cpu)
        assert torch.equal(torch.cuda.get_rng_state(), gpu)
    # the seed alone decides
    one, r1 = train_placement(**kw)
    torch.rand(7)
    two, r2 = train_placement(**kw)
    assert r1 == r2 and all(torch.equal(a, b) for a, b in zip(one.parameters(), two.parameters()))
