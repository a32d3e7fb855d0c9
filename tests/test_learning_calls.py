"""Calls of the policy operators (mobile_env.learning) that are refused rather than answered wrongly,
and calls as the documents show them."""
import pytest
import torch
from torch.autograd import forward_ad

gpu = pytest.mark.gpu


def _inputs(dev="cpu"):
    """What each operator is called with, float tensors first."""
    z = lambda *s: torch.zeros(*s, device=dev)
    return {
        "policy_loss": (dict(logits=z(4, 5), old_logp=z(4), advantage=z(4), weight=z(4) + 0.25,
                             ref_logp=z(4), action=torch.zeros(4, dtype=torch.int64, device=dev)),
                        ("logits", "old_logp", "advantage", "weight", "ref_logp")),
        "action_logp": (dict(logits=z(4, 5), action=torch.zeros(4, dtype=torch.int64, device=dev)),
                        ("logits",)),
        "advantages": (dict(reward=z(3, 4), done=torch.zeros(3, 4, dtype=torch.uint8, device=dev),
                            value=z(3, 4), last_value=z(4)), ("reward", "value", "last_value")),
        "clip_grad_norm": (dict(grads=z(6), max_norm=1.0, out=z(6)), ("grads", "out")),
    }


TANGENTS = [(op, name) for op, (_, names) in _inputs().items() for name in names]


def _check_tangent(op, name, dev):
    from mobile_env import learning
    kw, _ = _inputs(dev)[op]
    with forward_ad.dual_level():
        kw[name] = forward_ad.make_dual(kw[name], torch.ones_like(kw[name]))
        assert not kw[name].requires_grad
        with pytest.raises(RuntimeError, match="forward-mode"):
            getattr(learning, op)(**kw)


@pytest.mark.parametrize("op,name", TANGENTS)
def test_forward_mode_is_refused(op, name):
    """A dual number made of an ordinary tensor: it does not require a gradient."""
    _check_tangent(op, name, "cpu")


@gpu
@pytest.mark.parametrize("op,name", TANGENTS)
def test_forward_mode_is_refused_on_the_gpu(op, name):
    _check_tangent(op, name, "cuda")
