"""Policy operators on the GPU: what a policy over this engine's rollouts and station layouts is
trained and asked with, as hand-written kernels of libmev.so (include/mev.h, mev_policy_rows,
mev_advantages_run, mev_clip_norm).

* :func:`action_logp` -- log-probability of the taken action and entropy of every row of logits:
  what a rollout keeps as ``old_logp`` (or a reference policy as ``ref_logp``), one row or many.
* :func:`policy_loss` -- the clipped policy loss with a KL term towards a reference policy and an
  entropy bonus, differentiable in the logits.
* :func:`advantages` -- generalised advantages and returns, straight from the buffers of
  ``StepEngine.rollout`` (the multi-agent reward is the strided view ``obs[..., 3]``).
* :func:`clip_grad_norm` -- the global norm over many gradients, and the gradients clipped to it.

Every call runs on the current stream of its tensors' device, is asynchronous (nothing waits for
the GPU), can be captured into a HIP graph, and takes its buffers from torch's allocator, so
calls on several streams or in several graphs share nothing. Tensors that were written on another
stream need the usual ``wait_stream`` / ``record_stream``. There is no CPU fallback. Inputs with
forward-mode tangents are refused, and so are calls under a tracer or transform (``torch.jit.trace``,
``make_fx``, ``torch.export``, ``torch.func``; ``torch.compile`` runs them outside its graphs): they
would see the buffers without the work that fills them.

A backward pass is captured into a graph with no eager autograd graph of the same leaf parameters
alive (delete the eager loss first), as for every torch operator.
"""
from __future__ import annotations

from typing import Iterable, NamedTuple, Optional, Sequence, Tuple

import torch

from .core import _native as N

__all__ = ["PolicyLoss", "action_logp", "advantages", "clip_grad_norm", "policy_loss"]


class PolicyLoss(NamedTuple):
    """loss: float32 scalar (differentiable in the logits); logp, entropy: float32, one per row
    (0 in rows of weight 0; not differentiable)."""
    loss: torch.Tensor
    logp: torch.Tensor
    entropy: torch.Tensor


def action_logp(logits, action) -> Tuple[torch.Tensor, torch.Tensor]:
    """(log softmax(logits)[action], entropy of softmax(logits)), float32, one per row.

    logits [..., actions] float32 / bfloat16 / float16; action [...] int32 / int64. An action
    outside [0, actions) makes its row's log-probability NaN. Forbidden actions are logits of
    -inf; a row of nothing else has no distribution: log-probability -inf, entropy 0. No gradient
    flows (see :func:`policy_loss`)."""
    return N.torch_ops().action_logp(logits, action)


def policy_loss(logits, action, old_logp, advantage, weight=None, ref_logp=None, *,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                entropy_coef: float = 0.0) -> PolicyLoss:
    """The clipped policy loss of categorical logits. With L = log softmax(logits)[action], H the
    row's entropy, r = exp(L - old_logp) and d = ref_logp - L:

        loss = sum_i weight_i ( -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
                                + kl_coef (exp(d) - d - 1) - entropy_coef H )

    logits [..., actions] (float32 / bfloat16 / float16, any strides), action [...] int32 /
    int64; old_logp, advantage, weight, ref_logp: float32 [...], data (never differentiated).
    weight None: the mean over all rows. A padded row takes weight 0: it is not read, its outputs
    and gradient are 0 (weights of a masked mean: ``mask / mask.sum()``; over ranks: divided by
    the global sum). ref_logp None: no KL term. Forbidden actions are logits of -inf; a row of
    nothing else takes no part. An action outside [0, actions) makes the loss NaN.

    The gradient has the logits' dtype (rounded once) and is formed in the forward pass, for an
    incoming gradient of exactly one (``loss.backward()``); with any other the backward pass
    forms it anew, so a loss scale costs least inside the weights; so does a backward pass
    captured without its forward pass (capture both in one graph). Under saved-tensor hooks
    (``save_on_cpu``, checkpointing) the backward pass alone forms it, and nothing but the inputs is
    kept. Evaluate without gradients
    under ``torch.no_grad()``."""
    return PolicyLoss(*N.torch_ops().policy_loss(logits, action, old_logp, advantage, weight,
                                                 ref_logp, clip_low, clip_high, kl_coef,
                                                 entropy_coef))


def advantages(reward, done, value, last_value, gamma: float = 0.99, lam: float = 0.95,
               bootstrap_done: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """(advantages, returns) of a rollout, float32, in the reward's shape:

        delta_t = r_t + gamma V_{t+1} - V_t,  A_t = delta_t + gamma lam (1 - done_t) A_{t+1},
        returns_t = A_t + V_t,  V_T = last_value.

    reward float32 [T, E] or [T, E, U] (any strides: ``traj.reward``, ``traj.obs[..., 3]``);
    done uint8 / bool [T, E] (``traj.done``); value [T, E(, U)], the values of the observations
    the steps began with, and last_value [E(, U)], float32 / bfloat16 / float16 alike. A done
    step ends the trace. bootstrap_done (the default: this engine's episodes end by time limit,
    and the observation before the next step is the one the episode ended with) keeps V_{t+1} as
    that step's bootstrap; False takes 0. No gradient flows."""
    return N.torch_ops().advantages(reward, done, value, last_value, gamma, lam, bootstrap_done)


def clip_grad_norm(grads: Iterable[torch.Tensor], max_norm: float,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """The 2-norm over all elements of all ``grads`` (float32 scalar on their device; summed in
    64 bits), the gradients scaled by ``max_norm / norm`` where the norm is larger -- in place,
    or written to ``out`` (tensors of the same shapes, strides and dtypes; every element is
    written). A norm that is not finite scales nothing and is returned, so the caller can skip
    the step.

    grads: float32 / bfloat16 / float16 (mixed is fine) on one GPU, each filling one stretch of
    memory, none sharing memory with another; empty ones are skipped. Over
    ``[p.grad for p in policy.parameters() if p.grad is not None]``; a tensor counts as a list of
    itself."""
    grads, out = ([t] if isinstance(t, torch.Tensor) else t for t in (grads, out))
    return N.torch_ops().clip_grad_norm(list(grads), max_norm,
                                        None if out is None else list(out))
