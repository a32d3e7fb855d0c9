"""Station placement learned from the engine's reward.

The engine associates users by itself (base.py:236-241); what is left to decide is where the
stations stand, which chooseBaseStation.ipynb does by scoring random layouts (mobile_env.scoring).
Here a policy answers the users' positions with a cell for every station of every env, the engine
plays a step under those layouts, and the policy learns from the mean utility
(metrics.py:25-28) with the operators of :mod:`mobile_env.learning`: ``action_logp`` when it acts,
``advantages`` over the rollout, ``policy_loss`` and ``clip_grad_norm`` when it learns.

Scenario: MComCustom's (7 users at velocity 10, 5 to 10 stations, custom.py:16-18,68-77), the
number of stations drawn once per env; the rows behind an env's last station carry no weight.
"""
from __future__ import annotations

from typing import Dict, List, NamedTuple, Optional, Tuple

import torch

from .learning import action_logp, advantages, clip_grad_norm, policy_loss

__all__ = ["PlacementPolicy", "Rollout", "collect", "make_engine", "train_placement", "update"]

NUM_UES = 7


class PlacementPolicy(torch.nn.Module):
    """Users' positions [E, U, 2] in [0, 1] -> logits [E, stations, cells] and values [E]."""

    def __init__(self, stations: int, cells: int, num_ues: int = NUM_UES, hidden: int = 64):
        super().__init__()
        self.shape = (stations, cells)
        self.body = torch.nn.Linear(2 * num_ues, hidden)
        self.place = torch.nn.Linear(hidden, stations * cells)
        self.value = torch.nn.Linear(hidden, 1)

    def forward(self, positions):
        h = torch.tanh(self.body(positions.flatten(1)))
        return self.place(h).view(-1, *self.shape), self.value(h)[:, 0]


class Rollout(NamedTuple):
    """Leading axis: step. positions [T, E, U, 2], action [T, E, S] int64, logp [T, E, S],
    value [T, E], reward [T, E], done [T, E] uint8, last_value [E]; weight [E, S]."""
    positions: torch.Tensor
    action: torch.Tensor
    logp: torch.Tensor
    value: torch.Tensor
    reward: torch.Tensor
    done: torch.Tensor
    last_value: torch.Tensor
    weight: torch.Tensor


def make_engine(num_envs: int, stations: Tuple[int, int] = (5, 10), seed: int = 2024, device=None):
    """(engine, counts [E]): MComCustom's users under layouts that the policy will set."""
    from .core.engine import EngineParams, StepEngine
    from .scenarios.custom import MComCustom

    lo, most = stations
    if not 1 <= lo <= most:
        raise ValueError(f"stations must be (fewest, most) with 1 <= fewest <= most, got {stations}")
    cfg = MComCustom.default_config()
    g = torch.Generator().manual_seed(seed)
    count = torch.randint(lo, most + 1, (num_envs,), generator=g, dtype=torch.int32)
    xy = torch.randint(0, min(cfg["width"], cfg["height"]), (num_envs, most, 2), generator=g,
                       dtype=torch.int32)
    p = EngineParams(
        num_envs=num_envs, num_ues=NUM_UES, num_bs=most, width=cfg["width"], height=cfg["height"],
        ep_max_time=cfg["EP_MAX_TIME"], arrival_start=0,
        arrival_exit=cfg["arrival_params"]["ep_time"], first_step_active=True,
        movement_reseed=cfg["movement_params"].get("reset_rng_episode", True),
        velocity=cfg["ue"]["velocity"], bs=dict(cfg["bs"]),
        ue={k: cfg["ue"][k] for k in ("snr_tr", "noise", "height")})
    eng = StepEngine(p, xy, seed + torch.arange(num_envs).numpy(), bs_count=count.numpy(),
                     device=device)
    eng.reset()
    return eng, eng.bs_count


@torch.no_grad()
def collect(engine, policy, steps: int, cell: int, generator=None) -> Rollout:
    """``steps`` steps of every env, the stations placed anew before each (at cell centres).

    The engine resets an env whose episode is over at the start of its next step; here it is reset
    before the policy looks, so every action is played on the positions it was chosen for. What
    follows an episode's last step is then the next episode's first state: its value is that
    step's bootstrap (``last_value`` likewise), and the trace ends with the episode. Afterwards
    finished envs stand at their next episode's start, their ``done`` cleared."""
    if cell < 1:
        raise ValueError(f"cell must be at least 1, got {cell}")
    if steps < 1:
        raise ValueError(f"steps must be at least 1, got {steps}")
    S = engine.bs_xy.shape[1]
    columns = -(-int(engine.p.width) // cell)
    limit = torch.tensor([engine.p.width - 1, engine.p.height - 1], device=engine.device)
    keep = torch.arange(S, device=engine.device) < engine.bs_count[:, None]
    out: Dict[str, List[torch.Tensor]] = {k: [] for k in Rollout._fields[:6]}
    engine.reset(engine.done.clone())
    for _ in range(steps):
        positions = engine.obs[..., :2].clone()
        logits, value = policy(positions)
        # the largest of the logits plus Gumbel noise falls as softmax(logits) does
        u = torch.rand(logits.shape, device=logits.device, generator=generator)
        action = (logits.float() - (-(u.clamp_min(1e-20)).log()).log()).argmax(-1)
        logp, _ = action_logp(logits, action)
        xy = torch.stack([action % columns, action // columns], -1) * cell + cell // 2
        engine.set_bs_layout(torch.minimum(xy, limit).to(torch.int32))
        engine.step()
        for k, v in (("positions", positions), ("action", action), ("logp", logp),
                     ("value", value.float()), ("reward", engine.reward.clone()),
                     ("done", engine.done.clone())):
            out[k].append(v)
        engine.reset(out["done"][-1])
    last = policy(engine.obs[..., :2])[1].float()
    weight = keep.float()
    return Rollout(*(torch.stack(out[k]) for k in Rollout._fields[:6]), last, weight)


def update(policy, optimizer, rollout: Rollout, *, gamma: float = 0.9, lam: float = 0.95,
           clip: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.001,
           value_coef: float = 0.5, max_grad_norm: float = 0.5, ref_logp=None) -> Dict:
    """One pass of the policy over a rollout: the clipped loss of its placements, the squared
    error of its values, one step of the optimizer behind the clipped gradient. ``ref_logp``
    [T, E, S]: log-probabilities of a reference policy for the KL term."""
    T, E, S = rollout.action.shape
    adv, returns = advantages(rollout.reward, rollout.done, rollout.value, rollout.last_value,
                              gamma, lam)
    if adv.numel() > 1:  # (one alone has no deviation)
        adv = (adv - adv.mean()) / (adv.std() + 1e-6)
    weight = rollout.weight.expand(T, E, S)
    weight = weight / weight.sum()
    logits, value = policy(rollout.positions.flatten(0, 1))
    out = policy_loss(logits.view(T, E, S, -1), rollout.action, rollout.logp,
                      adv[..., None].expand(T, E, S), weight=weight, ref_logp=ref_logp,
                      clip_low=clip, clip_high=clip, kl_coef=kl_coef, entropy_coef=entropy_coef)
    value_loss = (value.view(T, E).float() - returns).square().mean()
    optimizer.zero_grad(set_to_none=True)
    (out.loss + value_coef * value_loss).backward()
    norm = clip_grad_norm([p.grad for p in policy.parameters() if p.grad is not None],
                          max_grad_norm)
    optimizer.step()
    return {"loss": out.loss.detach(), "value_loss": value_loss.detach(), "grad_norm": norm,
            "entropy": (out.entropy * weight).sum()}


def train_placement(num_envs: int = 1024, stations: Tuple[int, int] = (5, 10), cell: int = 10,
                    iterations: int = 20, steps: int = 20, epochs: int = 4, lr: float = 1e-3,
                    seed: int = 2024, device=None, policy: Optional[PlacementPolicy] = None,
                    **kw) -> Tuple[PlacementPolicy, List[float]]:
    """Learn to place stations: ``iterations`` rollouts of ``steps`` steps (20: an episode), each
    passed over ``epochs`` times (keywords of :func:`update`). Returns the policy and the mean
    reward of every rollout."""
    if cell < 1:
        raise ValueError(f"cell must be at least 1, got {cell}")
    eng, _ = make_engine(num_envs, stations, seed, device)
    cells = -(-int(eng.p.width) // cell) * -(-int(eng.p.height) // cell)
    if policy is None:
        with torch.random.fork_rng(devices=[]):  # (the caller's generators stay as they are)
            torch.default_generator.manual_seed(seed)
            policy = PlacementPolicy(stations[1], cells)
    policy = policy.to(eng.device)
    optimizer = torch.optim.Adam(policy.parameters(), lr=lr)
    g = torch.Generator(device=eng.device).manual_seed(seed)
    rewards = []
    for _ in range(iterations):
        rollout = collect(eng, policy, steps, cell, g)
        rewards.append(float(rollout.reward.mean()))
        for _ in range(epochs):
            update(policy, optimizer, rollout, **kw)
    eng.close()
    return policy, rewards
