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
stream need the usual ``wait_stream`` / ``record_stream``. There is no CPU fallback.

A backward pass is captured into a graph with no eager autograd graph of the same leaf parameters
alive (delete the eager loss first), as for every torch operator.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Iterable, NamedTuple, Optional, Sequence, Tuple

import torch

from .core import _native as N

__all__ = ["PolicyLoss", "action_logp", "advantages", "clip_grad_norm", "policy_loss"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # MEV_F32 / BF16 / F16


class PolicyLoss(NamedTuple):
    """loss: float32 scalar (differentiable in the logits); logp, entropy: float32, one per row
    (0 in rows of weight 0; not differentiable)."""
    loss: torch.Tensor
    logp: torch.Tensor
    entropy: torch.Tensor


def _stream(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _tensor(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.layout != torch.strided:
        raise ValueError(f"{name} must be a dense tensor")


def _on_gpu(t, name):
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} must live on a ROCm GPU (no CPU fallback)")


def _number(v, name, lo=-math.inf, hi=math.inf):
    v = float(v)
    if not (math.isfinite(v) and lo <= v <= hi):
        raise ValueError(f"{name} must be finite and lie in [{lo}, {hi}], got {v}")
    return v


def _logits(logits):
    _tensor(logits, "logits")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1 or logits.shape[-1] >= 2 ** 31:
        raise ValueError(f"logits must be [..., actions] with 1 to 2^31 - 1 actions, got "
                         f"{tuple(logits.shape)}")


def _action(action, logits):
    _tensor(action, "action")
    if action.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"action must be int32 or int64, got {action.dtype}")
    _like(action, "action", logits)
    return action.contiguous()


def _like(t, name, logits):
    if t.shape != logits.shape[:-1]:
        raise ValueError(f"{name} must have the logits' leading shape "
                         f"{tuple(logits.shape[:-1])}, got {tuple(t.shape)}")
    if t.device != logits.device:
        raise ValueError(f"{name} is on {t.device}, the logits are on {logits.device}")


def _row(t, name, logits):
    """One float32 number a row: data of the loss, never differentiated."""
    if t is None:
        return None
    _tensor(t, name)
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    _like(t, name, logits)
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} is data of the loss: no gradient reaches it (detach it)")
    return t.detach().contiguous()


def _rows_of(logits):
    """logits as rows in at most two strides: (tensor, rows, inner, outer stride, inner stride).
    Row i starts at element (i // inner) * outer + (i % inner) * inner stride. Logits whose
    actions are not adjacent, or whose leading axes need more strides, are copied once."""
    V = logits.shape[-1]
    if logits.stride(-1) != 1 and V > 1:
        logits = logits.contiguous()
    axes = []  # (size, stride), inner axis first, adjacent axes merged
    for n, s in zip(reversed(logits.shape[:-1]), reversed(logits.stride()[:-1])):
        if n == 1:
            continue
        if axes and s == axes[-1][0] * axes[-1][1]:
            axes[-1] = (axes[-1][0] * n, axes[-1][1])
        else:
            axes.append((n, s))
    if len(axes) > 2:
        return _rows_of(logits.contiguous())
    rows = math.prod(logits.shape[:-1])
    axes += [(1, 0)] * (2 - len(axes))
    return logits, rows, max(axes[0][0], 1), axes[1][1], axes[0][1]


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _launch(logits, action, old_logp=None, advantage=None, weight=None, ref_logp=None,
            coefs=(0.0, 0.0, 0.0, 0.0), outputs=True, loss=False, grad=None, scale=None,
            skip_unit=False):
    """One mev_policy_rows call; returns (loss, logp, entropy) as asked."""
    x, rows, inner, outer_stride, inner_stride = _rows_of(logits)
    kw = dict(dtype=torch.float32, device=logits.device)
    logp = torch.empty(logits.shape[:-1], **kw) if outputs else None
    ent = torch.empty(logits.shape[:-1], **kw) if outputs else None
    total = torch.empty((), **kw) if loss else None
    a = N.MevPolicy(
        logits=x.data_ptr(), action=action.data_ptr(), old_logp=_ptr(old_logp),
        advantage=_ptr(advantage), weight=_ptr(weight), ref_logp=_ptr(ref_logp),
        logp=_ptr(logp), entropy=_ptr(ent), loss=_ptr(total), grad=_ptr(grad),
        grad_scale=_ptr(scale), rows=rows, inner=inner, outer_stride=outer_stride,
        inner_stride=inner_stride, actions=logits.shape[-1], dtype=_DTYPES[logits.dtype],
        action_bytes=action.element_size(), skip_unit_scale=int(skip_unit),
        clip_low=coefs[0], clip_high=coefs[1], kl_coef=coefs[2], entropy_coef=coefs[3])
    L = N.lib()
    with torch.cuda.device(logits.device):
        need = L.mev_policy_workspace(C.byref(a))
        N.check(min(need, 0), "mev_policy_workspace")
        if need:
            work = torch.empty((need,), dtype=torch.uint8, device=logits.device)
            a.workspace, a.workspace_bytes = work.data_ptr(), need
        N.check(L.mev_policy_rows(C.byref(a), _stream(logits.device)), "mev_policy_rows")
    return total, logp, ent


def action_logp(logits, action) -> Tuple[torch.Tensor, torch.Tensor]:
    """(log softmax(logits)[action], entropy of softmax(logits)), float32, one per row.

    logits [..., actions] float32 / bfloat16 / float16; action [...] int32 / int64. An action
    outside [0, actions) makes its row's log-probability NaN. Forbidden actions are logits of
    -inf; a row of nothing else has no distribution: log-probability -inf, entropy 0. No gradient
    flows (see :func:`policy_loss`)."""
    _logits(logits)
    action = _action(action, logits)
    _on_gpu(logits, "logits")
    _, logp, ent = _launch(logits.detach(), action)
    return logp, ent


class _PolicyLoss(torch.autograd.Function):
    """The forward launch forms the gradient for an incoming gradient of one from the row it has
    at hand (one pass over the logits for both); the backward launch finds that on the device and
    leaves it, or forms it anew with the incoming gradient."""

    @staticmethod
    def forward(ctx, logits, action, old_logp, advantage, weight, ref_logp, coefs):
        grad = None
        if ctx.needs_input_grad[0]:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            ctx.save_for_backward(logits, action, old_logp, advantage, weight, ref_logp)
            ctx.coefs = coefs
            ctx.formed = grad
        loss, logp, ent = _launch(logits, action, old_logp, advantage, weight, ref_logp, coefs,
                                  loss=True, grad=grad)
        ctx.mark_non_differentiable(logp, ent)
        ctx.set_materialize_grads(False)
        return loss, logp, ent

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _logp, _ent):
        if g is None:
            return (None,) * 7
        logits, action, old_logp, advantage, weight, ref_logp = ctx.saved_tensors
        # handed out once: a second backward over a retained graph forms its own
        grad, ctx.formed = ctx.formed, None
        formed = grad is not None
        if not formed:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        _launch(logits, action, old_logp, advantage, weight, ref_logp, ctx.coefs, outputs=False,
                grad=grad, scale=g, skip_unit=formed)
        return (grad,) + (None,) * 6


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
    forms it anew, so a loss scale costs least inside the weights. Evaluate without gradients
    under ``torch.no_grad()``."""
    _logits(logits)
    action = _action(action, logits)
    if old_logp is None or advantage is None:
        raise TypeError("old_logp and advantage are needed")
    rows = [_row(t, name, logits) for t, name in (
        (old_logp, "old_logp"), (advantage, "advantage"), (weight, "weight"),
        (ref_logp, "ref_logp"))]
    coefs = (_number(clip_low, "clip_low", 0.0, 1.0), _number(clip_high, "clip_high", 0.0),
             _number(kl_coef, "kl_coef"), _number(entropy_coef, "entropy_coef"))
    _on_gpu(logits, "logits")
    return PolicyLoss(*_PolicyLoss.apply(logits, action, *rows, coefs))


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
    for t, name in ((reward, "reward"), (done, "done"), (value, "value"),
                    (last_value, "last_value")):
        _tensor(t, name)
        if t.device != reward.device:
            raise ValueError(f"{name} is on {t.device}, reward on {reward.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} is data: no gradient reaches it (detach it)")
    if reward.dtype != torch.float32:
        raise TypeError(f"reward must be float32, got {reward.dtype}")
    if done.dtype not in (torch.uint8, torch.bool):
        raise TypeError(f"done must be uint8 or bool, got {done.dtype}")
    if value.dtype not in _DTYPES or last_value.dtype != value.dtype:
        raise TypeError("value and last_value must both be float32, bfloat16 or float16, got "
                        f"{value.dtype} and {last_value.dtype}")
    if reward.dim() not in (2, 3):
        raise ValueError(f"reward must be [T, E] or [T, E, U], got {tuple(reward.shape)}")
    for t, name, shape in ((value, "value", reward.shape), (done, "done", reward.shape[:2]),
                           (last_value, "last_value", reward.shape[1:])):
        if t.shape != shape:
            raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    gamma, lam = _number(gamma, "gamma", 0.0, 1.0), _number(lam, "lam", 0.0, 1.0)
    _on_gpu(reward, "reward")
    T, E = reward.shape[:2]
    U = reward.shape[2] if reward.dim() == 3 else 1
    adv, ret = (torch.empty(reward.shape, dtype=torch.float32, device=reward.device)
                for _ in range(2))

    def strides(t, n):
        return (C.c_int64 * n)(*(tuple(t.stride()) + (0,))[:n])
    a = N.MevAdvantages(
        reward=reward.data_ptr(), value=value.data_ptr(), last_value=last_value.data_ptr(),
        done=done.data_ptr(), advantage=adv.data_ptr(), returns=ret.data_ptr(), T=T, E=E, U=U,
        reward_stride=strides(reward, 3), value_stride=strides(value, 3),
        last_stride=strides(last_value, 2), done_stride=strides(done, 2),
        value_dtype=_DTYPES[value.dtype], bootstrap_done=int(bool(bootstrap_done)), gamma=gamma,
        lam=lam)
    with torch.cuda.device(reward.device):
        N.check(N.lib().mev_advantages_run(C.byref(a), _stream(reward.device)),
                "mev_advantages_run")
    return adv, ret


def _dense(t) -> bool:
    """The elements fill one stretch of memory, in any order of axes."""
    if t.is_contiguous():
        return True
    n = 1
    for s, size in sorted((s, size) for s, size in zip(t.stride(), t.shape) if size != 1):
        if s != n:
            return False
        n *= size
    return True


def clip_grad_norm(grads: Iterable[torch.Tensor], max_norm: float,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """The 2-norm over all elements of all ``grads`` (float32 scalar on their device; summed in
    64 bits), the gradients scaled by ``max_norm / norm`` where the norm is larger -- in place,
    or written to ``out`` (tensors of the same shapes, strides and dtypes; every element is
    written). A norm that is not finite scales nothing and is returned, so the caller can skip
    the step.

    grads: float32 / bfloat16 / float16 (mixed is fine) on one GPU, each filling one stretch of
    memory, none sharing memory with another; empty ones are skipped. Over
    ``[p.grad for p in policy.parameters() if p.grad is not None]``."""
    grads = list(grads)
    if not grads:
        raise ValueError("no gradients")
    max_norm = _number(max_norm, "max_norm", 0.0)
    dst = grads if out is None else list(out)
    if len(dst) != len(grads):
        raise ValueError(f"out has {len(dst)} tensors for {len(grads)} gradients")
    device = None
    for g, o in zip(grads, dst):
        _tensor(g, "every gradient")
        if device is None:
            device = g.device
        if g.dtype not in _DTYPES:
            raise TypeError(f"gradients must be float32, bfloat16 or float16, got {g.dtype}")
        if g.device != device:
            raise ValueError(f"gradients on {g.device} and {device}")
        if not _dense(g):
            raise ValueError("a gradient must fill one stretch of memory (contiguous, or its axes "
                             "in another order)")
        if o is not g:
            _tensor(o, "out")
            if o.shape != g.shape or o.stride() != g.stride() or o.dtype != g.dtype or \
                    o.device != device:
                raise ValueError("out must match its gradient's shape, strides, dtype and device")
        if o.requires_grad and torch.is_grad_enabled():
            raise ValueError("a tensor that requires a gradient cannot be written")
    _on_gpu(grads[0], "every gradient")
    n = len(grads)
    src = (C.c_void_p * n)(*[g.data_ptr() for g in grads])
    to = (C.c_void_p * n)(*[o.data_ptr() for o in dst])
    numel = (C.c_int64 * n)(*[g.numel() for g in grads])
    dtype = (C.c_int32 * n)(*[_DTYPES[g.dtype] for g in grads])
    L = N.lib()
    with torch.cuda.device(device):
        need = L.mev_clip_norm_workspace(numel, n)
        N.check(min(need, 0), "mev_clip_norm_workspace")
        work = torch.empty((need,), dtype=torch.uint8, device=device)
        norm = torch.empty((), dtype=torch.float32, device=device)
        code = L.mev_clip_norm(src, to, numel, dtype, n, max_norm, norm.data_ptr(),
                               work.data_ptr(), need, _stream(device))
        if code == N.MEV_EINVAL:
            raise ValueError("gradients (or out) share memory")
        N.check(code, "mev_clip_norm")
    torch.autograd.graph.increment_version(dst)
    return norm
