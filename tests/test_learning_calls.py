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


# -- tracers and transforms ------------------------------------------------------------------------
def _traced(how, op, dev):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from mobile_env import learning
    kw, names = _inputs(dev)[op]
    first = names[0]

    def call(t):
        out = getattr(learning, op)(**{**kw, first: t})
        return out if isinstance(out, torch.Tensor) else out[0]
    x = kw[first]
    if how == "jit":
        torch.jit.trace(call, (x,), check_trace=False)
    elif how == "fx":
        make_fx(call)(x)
    elif how == "fx fake":
        make_fx(call, tracing_mode="fake")(x)
    elif how == "fx before dispatch":
        make_fx(call, pre_dispatch=True)(x)
    elif how == "fake":
        with FakeTensorMode() as mode:
            call(mode.from_tensor(x))
    elif how == "fake mode only":
        with FakeTensorMode():
            call(x)
    elif how == "fake tensor only":
        with FakeTensorMode() as mode:
            f = mode.from_tensor(x)
        call(f)
    elif how == "functionalize":
        torch.func.functionalize(call)(x)
    elif how == "vmap":
        torch.func.vmap(call)(torch.stack([x, x]))
    elif how == "grad":
        torch.func.grad(call)(x)
    elif how == "jvp":
        torch.func.jvp(call, (x,), (x,))


HOW = ["jit", "fx", "fx fake", "fx before dispatch", "fake", "fake mode only", "fake tensor only",
       "functionalize", "vmap", "grad", "jvp"]


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("op", list(_inputs()))
def test_tracing_is_refused(op, how):
    """A trace would hold the outputs' buffers and nothing that fills them."""
    with pytest.raises(RuntimeError, match="cannot be traced"):
        _traced(how, op, "cpu")


@gpu
@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("op", list(_inputs()))
def test_tracing_is_refused_on_the_gpu(op, how):
    with pytest.raises(RuntimeError, match="cannot be traced"):
        _traced(how, op, "cuda")


@gpu
def test_calls_under_a_counting_mode():
    """A dispatch mode that only looks on (no tracer) leaves the operators' results alone."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from mobile_env.learning import action_logp

    class Count(TorchDispatchMode):
        n = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.n += 1
            return func(*args, **(kwargs or {}))
    x = torch.randn(6, 9, device="cuda")
    a = torch.arange(6, device="cuda")
    want = action_logp(x, a)
    with Count() as mode:
        got = action_logp(x, a)
    assert mode.n and all(torch.equal(g, w) for g, w in zip(got, want))


# -- the documents' example ------------------------------------------------------------------------
def _examples():
    """Python blocks of the repository's documents that use the operators."""
    import glob
    import os
    import re
    from conftest import ROOT
    text = "\n".join(open(f, encoding="utf-8").read() for f in sorted(glob.glob(os.path.join(ROOT, "*.md"))))
    return [b for b in re.findall(r"```python\n(.*?)```", text, re.S)
            if "from mobile_env.learning import" in b]


def test_documents_have_an_example():
    assert len(_examples()) == 1


@gpu
def test_the_documents_example_runs():
    import mobile_env
    T, E, S, cells = 20, 6, 3, 50
    env = mobile_env.make("mobile-large-ma-v0", num_envs=E, seed=5)
    env.reset()
    traj = env.engine.rollout(T)
    g = torch.Generator().manual_seed(2)

    class Policy(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.head = torch.nn.Linear(60, S * cells + 1)

        def forward(self, obs):
            y = self.head(obs[..., :2].flatten(-2))  # (positions: the rates are bits a second)
            return y[..., 1:].reshape(*obs.shape[:2], S, cells), y[..., 0]
    policy = Policy().cuda()
    rows = lambda scale=1.0: (torch.randn(T, E, S, generator=g) * scale).cuda()
    names = dict(
        policy=policy, obs=traj.obs, traj=traj, T=T, E=E, S=S,
        action=torch.randint(0, cells, (T, E, S), generator=g).cuda(),
        last_value=policy(traj.obs[-1:])[1][0], value_ma=rows()[..., :1].expand(T, E, 30),
        last_ma=rows()[0, :, :1].expand(E, 30), old_logp=rows(0.1) - 4.0, ref_logp=rows(0.1) - 4.0,
        mask=torch.ones(T, E, S, device="cuda"))
    assert names["last_value"].requires_grad
    exec(_examples()[0], names)
    norm = sum(float(p.grad.double().square().sum()) for p in policy.parameters()) ** 0.5
    assert all(torch.isfinite(p.grad).all() for p in policy.parameters())
    assert 0.0 < norm <= 0.5 * (1 + 1e-5) and float(names["norm"]) >= norm * (1 - 1e-5)
    assert names["adv_ma"].shape == (T, E, 30) and names["returns"].shape == (T, E)
    env.close()


# -- what the loss keeps for its backward pass -----------------------------------------------------
def _loss_inputs(V=300, seed=3):
    g = torch.Generator().manual_seed(seed)
    r = lambda s=1.0: (torch.randn(40, 7, generator=g) * s).cuda()
    x = torch.randn(40, 7, V, generator=g).cuda()
    a = torch.randint(0, V, (40, 7), generator=g).cuda()
    old = torch.log_softmax(x, -1).gather(-1, a[..., None])[..., 0] - r(0.1)
    return x, (a, old, r()), dict(ref_logp=old + r(0.1), kl_coef=0.05, entropy_coef=0.01)


def _allocated(fn):
    """Bytes that fn took from the allocator, freed again or not."""
    key = "allocated_bytes.all.allocated"
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()[key]
    out = fn()
    torch.cuda.synchronize()
    return out, torch.cuda.memory_stats()[key] - before


@gpu
@pytest.mark.parametrize("scale", [1.0, 3.0])
def test_logits_of_odd_strides_are_copied_once(scale):
    """Logits whose actions are not adjacent: copied by the forward pass, and not again."""
    from mobile_env.learning import policy_loss
    x, args, kw = _loss_inputs()
    want, = torch.autograd.grad(policy_loss(y := x.clone().requires_grad_(), *args, **kw).loss * scale, y)
    odd = x.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    assert odd.stride(-1) == 7
    size = x.numel() * 4
    out, took = _allocated(lambda: policy_loss(odd, *args, **kw).loss * scale)
    assert 2 * size <= took < 3 * size  # the copy and the gradient
    (g,), took = _allocated(lambda: torch.autograd.grad(out, odd))
    # the gradient of another incoming one; a gradient of one is at hand
    assert took < (size if scale == 1.0 else 2 * size)
    assert torch.equal(g, want)


@gpu
def test_logits_of_odd_strides_under_saved_tensor_hooks():
    """A hook may give the copy back in any strides."""
    from mobile_env.learning import policy_loss
    x, args, kw = _loss_inputs()
    want, = torch.autograd.grad(policy_loss(y := x.clone().requires_grad_(), *args, **kw).loss, y)
    for v in (x, x.transpose(1, 2).contiguous().transpose(1, 2)):
        p = v.detach().requires_grad_()
        swap = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2) if t.dim() == 3 else t
        with torch.autograd.graph.saved_tensors_hooks(swap, lambda t: t):
            loss = policy_loss(p, *args, **kw).loss
        g, = torch.autograd.grad(loss, p)
        assert torch.equal(g, want)


@gpu
def test_what_saved_tensor_hooks_give_back_is_looked_at():
    """Other strides are taken as they are meant; another type, shape or device is refused before
    anything is launched."""
    from mobile_env.learning import policy_loss
    x, args, kw = _loss_inputs()
    kw["weight"] = torch.full((40, 7), 1 / 280, device="cuda")
    want, = torch.autograd.grad(policy_loss(y := x.clone().requires_grad_(), *args, **kw).loss, y)

    def grad(unpack, scale=1.0):
        p = x.clone().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
            loss = policy_loss(p, *args, **kw).loss
        return torch.autograd.grad(loss * scale, p)[0]
    gaps = lambda t: torch.stack([t, t], -1)[..., 0]
    assert not gaps(x).is_contiguous()
    assert torch.equal(grad(gaps), want)
    assert torch.equal(grad(lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)), want)
    for dims in (2, 3):  # the logits, or what stands beside them
        for bad in (lambda t: t.double(), lambda t: t[:1], lambda t: t.cpu(),
                    lambda t: torch.cat([t, t], -1), lambda t: t[..., :-1]):
            for scale in (1.0, 2.0):
                with pytest.raises((RuntimeError, TypeError, ValueError)):
                    grad(lambda t: bad(t) if t.dim() == dims else t, scale)


@gpu
def test_saved_tensor_hooks_hold_no_gradient():
    """Offloaded or recomputed, a loss keeps nothing of the logits' size on the GPU until its
    backward pass, which gives the same gradient."""
    from torch.utils.checkpoint import checkpoint
    from mobile_env.learning import policy_loss
    x, args, kw = _loss_inputs(V=3000)
    size = x.numel() * 4
    y = x.clone().requires_grad_()
    want, = torch.autograd.grad(policy_loss(y, *args, **kw).loss, y)

    def held(fn):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = fn()
        torch.cuda.synchronize()
        return out, torch.cuda.memory_allocated() - before
    loss, bytes_ = held(lambda: policy_loss(y, *args, **kw).loss)
    assert size <= bytes_ < 1.5 * size  # (without hooks: the formed gradient)
    del loss

    def offloaded():
        with torch.autograd.graph.save_on_cpu():
            return policy_loss(y, *args, **kw).loss
    loss, bytes_ = held(offloaded)
    assert bytes_ < 0.5 * size
    assert torch.equal(torch.autograd.grad(loss, y, retain_graph=True)[0], want)
    assert torch.equal(torch.autograd.grad(loss, y)[0], want)
    loss, bytes_ = held(lambda: checkpoint(
        lambda t: policy_loss(t * 1.0, *args, **kw).loss, y, use_reentrant=False))
    assert bytes_ < 0.5 * size
    assert torch.equal(torch.autograd.grad(loss, y)[0], want)
