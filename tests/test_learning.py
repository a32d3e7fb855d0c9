"""Policy operators (mobile_env.learning) against plain implementations in 64 bits.

Tolerances are sums of rounding bounds, written down before the first run. u = 2^-24 is half a
float32 step relative to the value. For a row of V logits with log-sum-exp m + ln s:

* a term e^(x - m) is off by a few u plus u |x - m| from its rounded argument; weighted by the
  terms themselves |x - m| averages to D = ln s - H. A float32 sum adds u a level; the longest
  chain here is one thread's V / 64 terms (rows in one wavefront) and the joins behind it:
  s is off by u (8 + 4 D + chain), chain = min(V, 64 + V / 64) + 16.
* logp = (x_a - m) - ln s adds 4 u (|x_a - m| + |ln s|); the entropy ln s - t / s carries the same
  chain once more on t / s = D.
* what follows is first-order: the ratio's relative error is logp's, the gradient's that of
  p and of its coefficient, and then half a step of the gradient's own type.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LO, HI = 0.8, 1.2
gpu = pytest.mark.gpu


# -- oracles -------------------------------------------------------------------------------------
def rows64(x, a):
    """(logp, entropy, p, log p) of rows in float64; a row of -inf only: -inf, 0, 0, 0."""
    x = x.double()
    none = (x == -math.inf).all(-1, keepdim=True)
    m = torch.where(none, torch.zeros_like(x[..., :1]), x.amax(-1, keepdim=True))
    d = x - m  # first: a row far from 0 keeps its differences
    lp = torch.where(none, torch.full_like(x, -math.inf), d - d.exp().sum(-1, keepdim=True).log())
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, torch.where(torch.isnan(p), p, torch.zeros_like(p)))
    return lp.gather(-1, a.long()[..., None])[..., 0], -plp.sum(-1), p, lp


def policy64(x, a, old, adv, w=None, ref=None, lo=LO, hi=HI, kl=0.0, ent=0.0):
    """loss, logp, entropy, gradient and the tolerances of each, in float64."""
    L, H, p, lp = rows64(x, a)
    V = x.shape[-1]
    n = L.numel()
    w = torch.full_like(L, 1.0 / n) if w is None else w.double()
    none = L == -math.inf
    none &= (x == -math.inf).all(-1)
    on = (w != 0) & ~none
    zero = torch.zeros_like(L)
    Ls = torch.where(on, L, zero)
    r = (Ls - old.double()).exp()
    A = adv.double()
    one, two = r * A, r.clamp(lo, hi) * A
    l = -torch.minimum(one, two)
    c = torch.where(one <= two, -one, zero)
    if ref is not None:
        d = ref.double() - Ls
        l = l + kl * (torch.expm1(d) - d)
        c = c - kl * torch.expm1(d)
    l = l - ent * H
    loss = torch.where(on, w * l, zero).sum()
    hot = torch.nn.functional.one_hot(a.long(), V).double()
    plp = torch.where(p > 0, p * (lp + H[..., None]), torch.zeros_like(p))
    g = w[..., None] * (c[..., None] * (hot - p) + ent * plp)
    g = torch.where(on[..., None], g, torch.zeros_like(g))
    # tolerances
    xs = x.double()
    m = torch.where(on, xs.amax(-1), zero)
    lns = torch.where(on, torch.where(on[..., None], xs - m[..., None], 0.0).exp().sum(-1).log(),
                      zero)
    D = (lns - H).clamp(min=0)
    chain = min(V, 64 + V / 64) + 16
    rel_s = U * (8 + 4 * D + chain)
    xa = torch.where(on, L + lns, zero)  # x_a - m
    t_lp = rel_s + 4 * U * (xa.abs() + lns.abs())
    t_H = rel_s * (1 + D) + U * (8 + 4 * D + chain) * D + 4 * U * (lns + D)
    t_r = torch.expm1(t_lp + 4 * U * (Ls - old.double()).abs() + 4 * U)
    t_l = r * A.abs() * (t_r + 4 * U)
    t_c = t_l.clone()
    if ref is not None:
        t_d = t_lp + 2 * U * d.abs()
        t_l = t_l + abs(kl) * (torch.expm1(d).abs() * t_d + d.exp() * t_d ** 2
                               + 8 * U * (torch.expm1(d) - d))
        t_c = t_c + abs(kl) * (d.exp() * t_d + 4 * U * torch.expm1(d).abs())
    t_l = t_l + abs(ent) * (t_H + 4 * U * H) + 4 * U * l.abs()
    t_loss = (torch.where(on, w.abs() * t_l, zero)).sum() + 2 * U * loss.abs()
    alp = torch.where(p > 0, lp.abs(), torch.zeros_like(lp))
    t_p = t_lp[..., None] + 4 * U * (alp + lns[..., None].abs()) + 8 * U
    t_g = w[..., None].abs() * (
        t_c[..., None] * (hot + p) + c[..., None].abs() * (p * t_p + 2 * U * hot)
        + abs(ent) * p * ((alp + H[..., None]) * (t_p + 4 * U) + t_p + t_H[..., None]))
    t_g = t_g + 4 * U * g.abs()
    return (loss, torch.where(w != 0, torch.where(none, L, Ls), zero),
            torch.where(on, H, zero), g), (t_loss, t_lp, t_H, t_g)


def check(got, want, tol, name, dtype=None):
    got, want = got.detach().double().cpu(), want.cpu()
    tol = torch.as_tensor(tol).cpu() + torch.zeros_like(want)
    if dtype is not None:  # the last rounding: half a step, or half the smallest number
        f = torch.finfo(dtype)
        tol = tol * (1 + f.eps) + want.abs() * f.eps / 2 + f.smallest_normal * f.eps / 2
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    bad = ~(same | ((got - want).abs() <= tol))
    if bad.any():
        i = int(bad.reshape(-1).nonzero()[0])
        raise AssertionError(
            f"{name}: {int(bad.sum())} of {bad.numel()} off, first [{i}] got "
            f"{got.reshape(-1)[i].item()} want {want.reshape(-1)[i].item()} tol "
            f"{tol.reshape(-1)[i].item()}")


def make(shape, V, dtype, seed=0, spread=2.0, banned=0.0, kl=True, dev="cuda"):
    """Inputs whose ratios stay off the clipping borders (either side is right there)."""
    g = torch.Generator().manual_seed(1000 * seed + V)
    x = (torch.randn(*shape, V, generator=g) * spread)
    a = torch.randint(0, V, shape, generator=g)
    if banned:
        ban = torch.rand(*shape, V, generator=g) < banned
        ban.scatter_(-1, a[..., None], False)
        x = x.masked_fill(ban, -math.inf)
    x = x.to(DT[dtype])
    L = rows64(x, a)[0]
    moved = torch.randn(shape, generator=g) * 0.3
    for b in (math.log(LO), math.log(HI)):
        moved = torch.where((moved - b).abs() < 0.01, moved + 0.03, moved)
    old = (L - moved.double()).float()
    adv = torch.randn(shape, generator=g)
    ref = (L + 0.3 * torch.randn(shape, generator=g).double()).float() if kl else None
    t = [x, a, old, adv, ref]
    return [v.to(dev) if v is not None else None for v in t]


def run_policy(x, a, old, adv, w=None, ref=None, kl=0.05, ent=0.01, scale=None):
    from mobile_env.learning import policy_loss
    x = x.detach().requires_grad_()
    out = policy_loss(x, a, old, adv, weight=w, ref_logp=ref, kl_coef=kl if ref is not None else 0,
                      entropy_coef=ent)
    g, = torch.autograd.grad(out.loss if scale is None else out.loss * scale, x)
    return out, g


def check_policy(x, a, old, adv, w=None, ref=None, kl=0.05, ent=0.01, name=""):
    out, g = run_policy(x, a, old, adv, w, ref, kl, ent)
    cpu = [t.cpu() if t is not None else None for t in (x, a, old, adv, w, ref)]
    want, tol = policy64(*cpu, kl=kl if ref is not None else 0.0, ent=ent)
    assert g.dtype == x.dtype and g.shape == x.shape
    check(out.logp, want[1], tol[1], name + " logp")
    check(out.entropy, want[2], tol[2], name + " entropy")
    check(out.loss, want[0], tol[0], name + " loss")
    check(g, want[3], tol[3], name + " gradient", x.dtype)
    return out, g


# -- the oracle itself, on the CPU ----------------------------------------------------------------
@pytest.mark.parametrize("kl,ent", [(0.0, 0.0), (0.3, 0.0), (0.0, 0.2), (0.3, 0.2)])
def test_oracle_gradient_against_differences(kl, ent):
    x, a, old, adv, ref = make((6, 3), 11, "f32", seed=4, dev="cpu")
    w = torch.rand(6, 3, generator=torch.Generator().manual_seed(1))
    w[2, 1:] = 0
    x = x.double()
    g = policy64(x, a, old, adv, w, ref, kl=kl, ent=ent)[0][3]
    h = 1e-6
    gen = torch.Generator().manual_seed(2)
    for _ in range(5):
        v = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        up = policy64(x + h * v, a, old, adv, w, ref, kl=kl, ent=ent)[0][0]
        dn = policy64(x - h * v, a, old, adv, w, ref, kl=kl, ent=ent)[0][0]
        fd, an = float(up - dn) / (2 * h), float((g * v).sum())
        # truncation h^2 and cancellation 2^-52 / h of a loss of order one
        assert abs(fd - an) < 1e-8, (fd, an)


def test_oracle_agrees_with_autograd():
    x, a, old, adv, ref = make((5, 2), 7, "f32", seed=5, dev="cpu")
    x = x.double().requires_grad_()
    lp = torch.log_softmax(x, -1)
    L = lp.gather(-1, a[..., None])[..., 0]
    r = (L - old.double()).exp()
    l = -torch.minimum(r * adv, r.clamp(LO, HI) * adv)
    d = ref.double() - L
    l = l + 0.3 * (d.exp() - d - 1) + 0.2 * (lp.exp() * lp).sum(-1)
    l.mean().backward()
    want, _ = policy64(x.detach(), a, old, adv, None, ref, kl=0.3, ent=0.2)
    assert abs(l.mean().item() - float(want[0])) < 1e-12
    torch.testing.assert_close(x.grad, want[3], rtol=1e-10, atol=1e-13)


# -- refusals (CPU) -------------------------------------------------------------------------------
def _ok(**kw):
    a = dict(logits=torch.zeros(4, 5), action=torch.zeros(4, dtype=torch.int64),
             old_logp=torch.zeros(4), advantage=torch.zeros(4))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,err", [
    (dict(), RuntimeError),                                             # CPU tensors: no fallback
    (dict(logits=[1.0]), TypeError),
    (dict(logits=torch.zeros(4, 5, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(4, 0)), ValueError),
    (dict(logits=torch.zeros(())), ValueError),
    (dict(action=torch.zeros(4)), TypeError),
    (dict(action=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(action=torch.zeros(4, 1, dtype=torch.int64)), ValueError),
    (dict(old_logp=None), TypeError),
    (dict(old_logp=torch.zeros(4, dtype=torch.float64)), TypeError),
    (dict(advantage=torch.zeros(3)), ValueError),
    (dict(advantage=torch.zeros(4, requires_grad=True)), ValueError),
    (dict(weight=torch.ones(4, dtype=torch.bool)), TypeError),
    (dict(ref_logp=torch.zeros(4, 1)), ValueError),
    (dict(clip_low=-0.1), ValueError),
    (dict(clip_low=1.5), ValueError),
    (dict(clip_high=math.inf), ValueError),
    (dict(kl_coef=math.nan), ValueError),
    (dict(entropy_coef=math.inf), ValueError),
    (dict(logits=torch.zeros(4, 5).to_sparse()), ValueError),
])
def test_policy_loss_refusals(kw, err):
    from mobile_env.learning import policy_loss
    with pytest.raises(err):
        policy_loss(**_ok(**kw))


def test_action_logp_refusals():
    from mobile_env.learning import action_logp
    with pytest.raises(RuntimeError):
        action_logp(torch.zeros(4, 5), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(TypeError):
        action_logp(torch.zeros(4, 5), torch.zeros(4, dtype=torch.int16))
    with pytest.raises(ValueError):
        action_logp(torch.zeros(4, 5), torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("kw,err", [
    (dict(), RuntimeError),
    (dict(reward=torch.zeros(3, 4, dtype=torch.float64)), TypeError),
    (dict(reward=torch.zeros(3)), ValueError),
    (dict(done=torch.zeros(3, 4)), TypeError),
    (dict(done=torch.zeros(3, 5, dtype=torch.uint8)), ValueError),
    (dict(value=torch.zeros(4, 4)), ValueError),
    (dict(value=torch.zeros(3, 4, dtype=torch.float64)), TypeError),
    (dict(value=torch.zeros(3, 4, requires_grad=True)), ValueError),
    (dict(last_value=torch.zeros(4, dtype=torch.bfloat16)), TypeError),
    (dict(last_value=torch.zeros(3)), ValueError),
    (dict(gamma=1.1), ValueError),
    (dict(lam=-0.1), ValueError),
    (dict(lam=math.nan), ValueError),
])
def test_advantages_refusals(kw, err):
    from mobile_env.learning import advantages
    a = dict(reward=torch.zeros(3, 4), done=torch.zeros(3, 4, dtype=torch.bool),
             value=torch.zeros(3, 4), last_value=torch.zeros(4))
    a.update(kw)
    with pytest.raises(err):
        advantages(**a)


@pytest.mark.parametrize("grads,kw,err", [
    ([torch.zeros(3)], {}, RuntimeError),
    ([], {}, ValueError),
    ([None], {}, TypeError),
    ([torch.zeros(3, dtype=torch.float64)], {}, TypeError),
    ([torch.zeros(3)], dict(max_norm=-1.0), ValueError),
    ([torch.zeros(3)], dict(max_norm=math.inf), ValueError),
    ([torch.zeros(3)], dict(max_norm=1e39), ValueError),
    ([torch.zeros(4, 4)[:, ::2]], {}, ValueError),
    ([torch.zeros(1, 4).expand(3, 4)], {}, ValueError),
    ([torch.zeros(3)], dict(out=[]), ValueError),
    ([torch.zeros(3)], dict(out=[torch.zeros(4)]), ValueError),
    ([torch.zeros(3)], dict(out=[torch.zeros(3, dtype=torch.bfloat16)]), ValueError),
    ([torch.zeros(2, 3)], dict(out=[torch.zeros(3, 2).t()]), ValueError),
    ([torch.zeros(3, requires_grad=True)], {}, ValueError),
])
def test_clip_refusals(grads, kw, err):
    from mobile_env.learning import clip_grad_norm
    with pytest.raises(err):
        clip_grad_norm(grads, **{"max_norm": 1.0, **kw})


def test_c_abi_refuses_bad_arguments():
    """The C entries turn bad arguments into MEV_EINVAL before anything is launched."""
    from mobile_env.core import _native as N
    L = N.lib()
    fake = 1 << 20  # never read: every call below is refused
    base = dict(logits=fake, action=fake, logp=fake, entropy=fake, rows=4, inner=4,
                inner_stride=8, actions=8, dtype=0, action_bytes=8)

    def rc(**kw):
        a = N.MevPolicy(**{**base, **kw})
        return L.mev_policy_rows(C.byref(a), None)
    for kw in (dict(logits=None), dict(action=None), dict(rows=-1), dict(inner=0),
               dict(actions=0), dict(dtype=3), dict(action_bytes=2), dict(logp=None),
               dict(old_logp=fake), dict(loss=fake), dict(grad=fake),
               # many rows: a workspace is needed
               dict(rows=1 << 20, old_logp=fake, advantage=fake, loss=fake),
               dict(rows=1 << 20, old_logp=fake, advantage=fake, loss=fake, workspace=fake,
                    workspace_bytes=8),
               dict(skip_unit_scale=1), dict(skip_unit_scale=1, grad_scale=fake)):
        assert rc(**kw) == N.MEV_EINVAL, kw
    assert L.mev_policy_rows(None, None) == N.MEV_EINVAL
    assert L.mev_policy_workspace(None) == N.MEV_EINVAL
    a = N.MevAdvantages(T=2, E=2, U=1)
    assert L.mev_advantages_run(C.byref(a), None) == N.MEV_EINVAL
    a = N.MevAdvantages(T=0, E=2, U=1)
    assert L.mev_advantages_run(C.byref(a), None) == N.MEV_OK
    a = N.MevAdvantages(T=-1, E=2, U=1)
    assert L.mev_advantages_run(C.byref(a), None) == N.MEV_EINVAL

    def clip(ptrs, sizes, max_norm=1.0, dst=None, dtypes=None, ws=1 << 20):
        n = len(ptrs)
        num = (C.c_int64 * n)(*sizes)
        return L.mev_clip_norm((C.c_void_p * n)(*ptrs), (C.c_void_p * n)(*(dst or ptrs)), num,
                               (C.c_int32 * n)(*(dtypes or [0] * n)), n, max_norm, fake, fake, ws,
                               None)
    assert clip([fake], [-1]) == N.MEV_EINVAL
    assert clip([None], [4]) == N.MEV_EINVAL
    assert clip([fake], [4], max_norm=math.nan) == N.MEV_EINVAL
    assert clip([fake], [4], dtypes=[7]) == N.MEV_EINVAL
    assert clip([fake], [4], ws=4) == N.MEV_EINVAL
    assert clip([fake, fake + 12], [4, 4]) == N.MEV_EINVAL           # overlap
    assert clip([fake, fake], [4, 4]) == N.MEV_EINVAL                # the same twice
    assert clip([fake], [4], dst=[fake + 4]) == N.MEV_EINVAL         # shifted onto itself
    assert clip([fake, 2 * fake], [4, 4], dst=[2 * fake, fake]) == N.MEV_EINVAL


@pytest.mark.parametrize("kw", [dict(kl_coef=1e39), dict(kl_coef=-1e39), dict(entropy_coef=1e300)])
def test_policy_loss_refuses_coefficients_beyond_float32(kw):
    from mobile_env.learning import policy_loss
    with pytest.raises(ValueError):
        policy_loss(**_ok(**kw))


def test_c_abi_refuses_rows_beyond_any_buffer():
    """A count whose workspace would not fit 64 bits."""
    from mobile_env.core import _native as N
    a = N.MevPolicy(rows=1 << 62, inner=1, actions=8, dtype=0, action_bytes=8)
    assert N.lib().mev_policy_workspace(C.byref(a)) == N.MEV_EINVAL
    a.actions = 200000
    assert N.lib().mev_policy_workspace(C.byref(a)) == N.MEV_EINVAL
    a.rows = 1 << 40
    assert N.lib().mev_policy_workspace(C.byref(a)) > 0


def test_no_packed_float32_instructions():
    """Packed float32 arithmetic is kept out of the device code (csrc/Makefile, NOPK)."""
    import os
    import re
    import shutil
    import subprocess
    from conftest import ROOT
    if shutil.which("/opt/rocm/bin/hipcc") is None:
        pytest.skip("hipcc not available")
    d = os.path.join(ROOT, "mobile-env-gan_amd")
    subprocess.run(["make", "-C", os.path.join(d, "csrc"), "asm"], check=True,
                   stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    for f in ("mev_step-gfx950.s", "mev_learn-gfx950.s"):
        text = open(os.path.join(d, "lib", f)).read()
        assert not re.search(r"v_pk_(add|mul|fma)_f32", text), f


def test_host_code_under_asan(tmp_path):
    """The entries' host code under AddressSanitizer + UBSan (tests/asan/learn_driver.c)."""
    import os
    import shutil
    import subprocess
    from conftest import ROOT
    clang = "/opt/rocm/llvm/bin/clang"
    if not os.path.exists(clang) or shutil.which("make") is None:
        pytest.skip("ROCm clang / make not available")
    subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "mobile-env-gan_amd", "csrc"), "asan"],
                   check=True, timeout=900)
    lib = os.path.join(ROOT, "mobile-env-gan_amd", "lib", "libmev_asan.so")
    drv = str(tmp_path / "learn_driver")
    subprocess.run([clang, "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-g",
                    "-I", os.path.join(ROOT, "include"), "-o", drv,
                    os.path.join(ROOT, "tests", "asan", "learn_driver.c"), lib,
                    "-Wl,-rpath," + os.path.dirname(lib)], check=True, timeout=120)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:verify_asan_link_order=0",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1", HIP_VISIBLE_DEVICES="")
    r = subprocess.run([drv], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


# -- policy loss on the GPU -----------------------------------------------------------------------
# both sides of the shapes' limits, and between them
SIZES = [1, 2, 3, 4, 5, 7, 8, 9, 12, 13, 14, 16, 17, 20, 21, 24, 25, 31, 32, 33, 40, 63, 64, 65, 71,
         96, 97, 100, 127, 128, 129, 135, 192, 193, 200, 255, 256, 257, 263, 384, 385, 511, 512,
         513, 519, 768, 769, 1000, 1024, 1031, 1280, 1281, 1536, 1537, 2047, 2048, 2049, 2560, 2561,
         4096, 4099, 6144, 6145, 8191, 8192, 8193, 12288, 12289, 16384, 16391, 20480, 20481, 24576,
         24581, 32768, 32769, 40000, 40961, 41567, 49152, 49153, 65536, 65543, 98304, 98311, 131072,
         140003]


@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", SIZES)
def test_policy_loss_sizes(V, dtype):
    rows = 300 if V <= 257 else 37 if V < 5000 else 5
    x, a, old, adv, ref = make((rows,), V, dtype, banned=0.1 if V > 8 else 0.0)
    check_policy(x, a, old, adv, None, ref, name=f"V={V} {dtype}")
    from mobile_env.learning import action_logp
    want, tol = policy64(x.cpu(), a.cpu(), old.cpu(), adv.cpu())
    logp, ent = action_logp(x, a.int())
    check(logp, want[1], tol[1], "action_logp logp")
    check(ent, want[2], tol[2], "action_logp entropy")


# rows of 24 to 4,096 16-bit actions: what a row of 2 to 64 lanes and 2 to 8 vectors a lane holds
HELD = [8 * g * n for g, ns in ((1, (1, 2, 3)), (2, (2, 3)), (4, range(2, 9)), (8, range(5, 9)),
                                (16, range(5, 9)), (32, range(5, 9)), (64, (5, 7, 8)))
        for n in ns]


@gpu
@pytest.mark.parametrize("off", [-9, -7, -1, 0, 1, 2, 4])
@pytest.mark.parametrize("dtype", list(DT))
def test_policy_loss_borders_of_the_lanes(dtype, off):
    """Rows a little shorter and longer than what a number of lanes holds: the last vector then
    repeats elements of the one before. A row without weight, a forbidden action, one alone."""
    for full in HELD:
        V = (full if dtype != "f32" else full // 2) + off
        if V < 2:
            continue
        x, a, old, adv, ref = make((11,), V, dtype, seed=V)
        w = torch.rand(11, generator=torch.Generator().manual_seed(V)).cuda() / 11
        w[3] = 0.0
        x[4, torch.arange(V, device="cuda") != a[4]] = -math.inf
        x[5, V - 1] = x[5, V - 1] if int(a[5]) == V - 1 else -math.inf
        check_policy(x, a, old, adv, w, ref, name=f"{V} actions")


@gpu
@pytest.mark.parametrize("V", [65537, 98305, 114687, 114697, 131071, 131072, 131073])
@pytest.mark.parametrize("dtype", list(DT))
def test_policy_loss_rows_of_a_workgroup(dtype, V):
    """The longest rows that one workgroup holds, with enough of them to be given one each; most
    carry no weight, so that the oracle has little to do."""
    V = V if dtype != "f32" else (V + 1) // 2
    x, a, old, adv, ref = make((6,), V, dtype, seed=19)
    at = torch.tensor([0, 7, 63, 100, 150, 199], device="cuda")
    big = [torch.zeros((200,) + t.shape[1:], dtype=t.dtype, device="cuda")
           for t in (x, a, old, adv, ref)]
    for t, v in zip(big, (x, a, old, adv, ref)):
        t[at] = v
    w = torch.zeros(200, device="cuda")
    w[at] = torch.tensor([0.1, 0.3, 0.2, 0.1, 0.1, 0.2], device="cuda")
    out, g = run_policy(*big[:4], w, big[4])
    want, tol = policy64(x.cpu(), a.cpu(), old.cpu(), adv.cpu(), w[at].cpu(), ref.cpu(), kl=0.05,
                         ent=0.01)
    check(out.logp[at], want[1], tol[1], "logp")
    check(out.entropy[at], want[2], tol[2], "entropy")
    check(out.loss, want[0], tol[0], "loss")
    check(g[at], want[3], tol[3], "gradient", x.dtype)
    g[at] = 0
    assert not g.any() and not out.logp[w == 0].any() and not out.entropy[w == 0].any()


@gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 255, 257, 1023, 20001])
@pytest.mark.parametrize("V", [3, 14, 40, 130])
def test_policy_loss_row_counts(rows, V):
    x, a, old, adv, ref = make((rows,), V, "bf16", seed=2)
    w = torch.rand(rows, generator=torch.Generator().manual_seed(rows)) / rows
    w[::3] = 0
    check_policy(x, a, old, adv, w.cuda(), ref, name=f"rows={rows}")


@gpu
@pytest.mark.parametrize("V", [7, 13, 48, 515, 4099])
@pytest.mark.parametrize("dtype", list(DT))
def test_policy_loss_strides(V, dtype):
    """Padded rows, swapped leading axes, every other action, shared rows and offset views give
    what their contiguous copies give."""
    x, a, old, adv, ref = make((6, 5), V, dtype, seed=3)
    want, gw = run_policy(x, a, old, adv, None, ref)
    pad = torch.full((6, 5, V + 3), float("nan"), dtype=x.dtype, device="cuda")
    pad[..., 2:V + 2] = x
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)
    gaps = torch.full((6, 5, 2 * V), float("nan"), dtype=x.dtype, device="cuda")
    gaps[..., ::2] = x
    deep = torch.full((6, 2, 5, 2, V), float("nan"), dtype=x.dtype, device="cuda")
    deep[:, 1, :, 0] = x
    for name, v in (("padded", pad[..., 2:V + 2]), ("swapped", swapped), ("gaps", gaps[..., ::2]),
                    ("deep", deep[:, 1, :, 0])):
        assert torch.equal(v, x)
        out, g = run_policy(v, a, old, adv, None, ref)
        assert torch.equal(out.logp, want.logp), name
        assert torch.equal(out.loss, want.loss) and torch.equal(g, gw), name
    # side inputs with gaps
    side = [torch.stack([t, t], -1)[..., 0] for t in (a, old, adv, ref)]
    assert not side[0].is_contiguous()
    out, g = run_policy(x, side[0], side[1], side[2], None, side[3])
    assert torch.equal(out.loss, want.loss) and torch.equal(g, gw)
    # one row of logits shared by all rows: its gradient is the sum of theirs
    one = x[:1, :1].detach().requires_grad_()
    from mobile_env.learning import policy_loss
    out = policy_loss(one.expand(6, 5, V), a, old, adv, entropy_coef=0.01)
    g, = torch.autograd.grad(out.loss, one)
    rep = x[:1, :1].expand(6, 5, V).contiguous()
    w64, tol = policy64(rep.cpu(), a.cpu(), old.cpu(), adv.cpu(), ent=0.01)
    f = torch.finfo(x.dtype)
    # each of 30 summands rounded to its type, then their sum (torch: one rounding a partial sum)
    t = (tol[3] + w64[3].abs() * f.eps).sum((0, 1)) + 2 * f.smallest_normal
    check(g[0, 0], w64[3].sum((0, 1)), t + w64[3].abs().sum((0, 1)) * f.eps, "shared row")


@gpu
@pytest.mark.parametrize("V", [6, 14, 40, 300, 5000, 70001])
@pytest.mark.parametrize("dtype", list(DT))
def test_policy_loss_masks(V, dtype):
    """Rows without weight are not looked at; rows of -inf take no part; the type's lowest value
    and large offsets are ordinary logits; a forbidden action that was taken is -inf."""
    n = 12
    x, a, old, adv, ref = make((n,), V, dtype, seed=6)
    low = torch.finfo(x.dtype).min
    w = torch.full((n,), 1.0 / 8, device="cuda")
    x[1] = float("nan"); w[1] = 0
    x[2] = float("inf"); w[2] = 0
    old[3] = float("nan"); adv[3] = float("inf"); w[3] = 0
    x[4] = -math.inf
    x[5] = low
    x[6, :] = low
    x[6, a[6]] = 1.0
    x[7] = x[7] + (1000.0 if dtype != "f16" else 500.0)
    x[8, :] = -math.inf
    x[8, a[8]] = 0.0
    for i in (5, 6, 7, 8):
        L = rows64(x[i].cpu(), a[i].cpu())[0]
        old[i] = (L - 0.05).float(); ref[i] = (L + 0.1).float()
    a[1] = -1
    a[2] = V + 5
    a_ok = a.clone(); a_ok[1] = 0; a_ok[2] = 0
    xo = x.clone(); xo[1] = 0; xo[2] = 0
    oo, ao = old.clone(), adv.clone(); oo[3] = 0; ao[3] = 0
    want, tol = policy64(xo.cpu(), a_ok.cpu(), oo.cpu(), ao.cpu(), w.cpu(), ref.cpu(), kl=0.05,
                         ent=0.01)
    out, g = run_policy(x, a, old, adv, w, ref)
    check(out.logp, want[1], tol[1], "logp")
    check(out.entropy, want[2], tol[2], "entropy")
    check(out.loss, want[0], tol[0], "loss")
    check(g, want[3], tol[3], "gradient", x.dtype)
    assert (g[[1, 2, 3, 4]] == 0).all()


@gpu
@pytest.mark.parametrize("V", [9, 40, 700, 20000, 140003])
def test_policy_loss_bad_values_are_loud(V):
    """NaN logits, +inf logits and actions out of range give NaN in their row and the loss, and
    leave the other rows alone."""
    x, a, old, adv, ref = make((6,), V, "f32", seed=7)
    good, gg = run_policy(x, a, old, adv, None, ref)
    x[1, V // 2] = float("nan")
    x[2, V - 1] = float("inf")
    a[3], a[4] = V, -1
    out, g = run_policy(x, a, old, adv, None, ref)
    assert torch.isnan(out.loss)
    for i in (1, 2, 3, 4):
        assert torch.isnan(out.logp[i]) and torch.isnan(g[i]).all()
    for i in (0, 5):
        assert torch.equal(out.logp[i], good.logp[i]) and torch.equal(g[i], gg[i])


@gpu
@pytest.mark.parametrize("V", [5, 40, 700, 20000, 140003])
@pytest.mark.parametrize("dtype", list(DT))
def test_policy_loss_of_a_forbidden_action(V, dtype):
    """The taken action's logit is -inf now: log-probability -inf, ratio 0 -- the clipped branch
    where the advantage is negative -- and no gradient but the entropy's; an infinite loss where
    a KL term asks for it."""
    x, a, old, adv, ref = make((4,), V, dtype, seed=16)
    x.scatter_(1, a[:, None], -math.inf)
    adv.copy_(torch.tensor([1.0, -2.0, 0.0, 3.0]))
    out, g = run_policy(x, a, old, adv, None, None, ent=0.0)
    assert (out.logp == -math.inf).all() and torch.isfinite(out.entropy).all()
    # clip_low 0.2: 1 - 0.2 times 2, over four rows
    assert abs(float(out.loss) - (1 - 0.2) * 2.0 / 4) <= 0.4 * U and (g == 0).all()
    out, g = run_policy(x, a, old, adv, None, None, ent=0.01)
    w64, tol = policy64(x.cpu(), a.cpu(), old.cpu(), adv.cpu(), None, None, ent=0.01)
    assert torch.isfinite(g).all() and torch.isfinite(out.loss)
    H = out.entropy.double()
    assert abs(float(out.loss) - 0.4 + 0.01 * float(H.mean())) <= U * (1 + float(H.mean()))
    out, g = run_policy(x, a, old, adv, None, ref, kl=0.1)
    assert float(out.loss) == math.inf
    out, g = run_policy(x, a, old, adv, None, ref, kl=0.0, ent=0.0)  # a weight of 0: no term
    assert abs(float(out.loss) - 0.4) <= 0.4 * U and (g == 0).all()


@gpu
def test_policy_loss_ratios_far_from_one():
    """Ratios that overflow, vanish, or differ in the last place of a large log ratio."""
    x, a, old, adv, _ = make((12,), 30, "f32", seed=17)
    L = rows64(x.cpu(), a.cpu())[0]
    old.copy_((L - torch.tensor([200., -200., 60., -60., 20., -20., 5., -5., 88., -88., 1., 0.],
                                dtype=torch.float64)).float())
    for A in (1.0, -1.0):
        adv.fill_(A)
        # (row by row: the sum of an infinite and a finite one says nothing of the second)
        for i in range(12):
            s = slice(i, i + 1)
            out, g = run_policy(x[s], a[s], old[s], adv[s], None, None, ent=0.0)
            w64, tol = policy64(x[s].cpu(), a[s].cpu(), old[s].cpu(), adv[s].cpu())
            if abs(float(w64[0])) > 3e38:
                assert float(out.loss) == math.copysign(math.inf, float(w64[0]))
                continue
            # the loss is a float32 number; a float32 ratio below 2^-126 is 0 (the exponential has
            # no subnormal results), so its gradient is off by no more than that
            check(out.loss, w64[0], tol[0], f"loss {i} {A}", torch.float32)
            check(g, w64[3], tol[3] + 2.0 ** -126, f"gradient {i} {A}", torch.float32)


@gpu
def test_policy_loss_refuses_changed_logits_and_second_derivatives():
    from mobile_env.learning import policy_loss
    x, a, old, adv, _ = make((6,), 9, "f32", seed=18)
    p = x.clone().requires_grad_()
    y = p * 1.0
    out = policy_loss(y, a, old, adv)
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError):
        out.loss.backward()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(policy_loss(p, a, old, adv).loss, p, create_graph=True)
    assert p.grad is None


@gpu
def test_two_calls_at_once():
    """Two threads on streams of their own."""
    import threading
    data = [make((2000,), 300 + 7 * k, "bf16", seed=19 + k) for k in range(2)]
    want = [run_policy(*d[:4], None, d[4]) for d in data]
    torch.cuda.synchronize()
    got = [None, None]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k] = run_policy(*data[k][:4], None, data[k][4])
            torch.cuda.current_stream().synchronize()
    ts = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    for (o, g), (wo, wg) in zip(got, want):
        assert torch.equal(o.loss, wo.loss) and torch.equal(g, wg)


@gpu
@pytest.mark.parametrize("shape,V", [((0,), 5), ((3, 0), 40), ((), 17), ((1,), 1), ((2, 1, 3), 6)])
def test_policy_loss_small_shapes(shape, V):
    from mobile_env.learning import action_logp
    x, a, old, adv, ref = make(shape, V, "f32", seed=8)
    out, g = run_policy(x, a, old, adv, None, ref)
    assert out.logp.shape == shape and g.shape == x.shape and out.loss.shape == ()
    if 0 in shape:
        assert float(out.loss) == 0.0
    else:
        check_policy(x, a, old, adv, None, ref)
    assert action_logp(x, a)[0].shape == shape


@gpu
@pytest.mark.parametrize("V", [13, 300, 9000, 140003])
@pytest.mark.parametrize("dtype", list(DT))
def test_policy_loss_incoming_gradient(V, dtype):
    """An incoming gradient other than one, a second backward over a retained graph, and the
    no-gradient form."""
    from mobile_env.learning import policy_loss
    x, a, old, adv, ref = make((7,), V, dtype, seed=9)
    want, tol = policy64(x.cpu(), a.cpu(), old.cpu(), adv.cpu(), None, ref.cpu(), kl=0.05, ent=0.01)
    _, g = run_policy(x, a, old, adv, None, ref, scale=384.0)
    check(g, want[3] * 384, tol[3] * 384, "scaled", x.dtype)
    x.requires_grad_()
    out = policy_loss(x, a, old, adv, ref_logp=ref, kl_coef=0.05, entropy_coef=0.01)
    g1, = torch.autograd.grad(out.loss, x, retain_graph=True)
    keep = g1.clone()
    g2, = torch.autograd.grad(out.loss, x, retain_graph=True)
    g3, = torch.autograd.grad(out.loss * 2, x)
    assert g1.data_ptr() != g2.data_ptr() and torch.equal(g1, keep)
    assert torch.equal(g1, g2)
    check(g3, want[3] * 2, tol[3] * 2, "twice", x.dtype)
    with torch.no_grad():
        o2 = policy_loss(x, a, old, adv, ref_logp=ref, kl_coef=0.05, entropy_coef=0.01)
    assert not o2.loss.requires_grad and torch.equal(o2.loss, out.loss.detach())
    assert not out.logp.requires_grad and not out.entropy.requires_grad
    x.grad = None
    policy_loss(x, a, old, adv).loss.backward()
    policy_loss(x, a, old, adv).loss.backward()  # accumulates
    g0, = torch.autograd.grad(policy_loss(x, a, old, adv).loss, x)
    assert torch.equal(x.grad, g0 + g0)


@gpu
def test_policy_loss_gradient_against_differences():
    """The kernel's gradient against differences of the kernel's loss: truncation as the 64-bit
    oracle shows it at the same points, plus the loss's own rounding over the step."""
    x, a, old, adv, ref = make((8, 4), 37, "f32", seed=10, spread=1.0)
    out, g = run_policy(x, a, old, adv, None, ref, kl=0.3, ent=0.2)
    gen = torch.Generator().manual_seed(3)
    h = 2.0 ** -9
    cpu = [t.cpu() for t in (a, old, adv)]
    w64, tol = policy64(x.cpu(), *cpu, None, ref.cpu(), kl=0.3, ent=0.2)
    for _ in range(4):
        v = torch.randn(x.shape, generator=gen).cuda()
        hi, lo = x + h * v, x - h * v
        fd = float(run_policy(hi, a, old, adv, None, ref, 0.3, 0.2)[0].loss.double()
                   - run_policy(lo, a, old, adv, None, ref, 0.3, 0.2)[0].loss.double()) / (2 * h)
        wh, th = policy64(hi.cpu(), *cpu, None, ref.cpu(), kl=0.3, ent=0.2)
        wl, tl = policy64(lo.cpu(), *cpu, None, ref.cpu(), kl=0.3, ent=0.2)
        trunc = abs(float(wh[0] - wl[0]) / (2 * h) - float((w64[3] * v.cpu().double()).sum()))
        bound = trunc + float(th[0] + tl[0]) / (2 * h) + float((tol[3] * v.cpu().abs()).sum())
        assert abs(fd - float((g * v).double().sum())) <= bound + 1e-9, (fd, bound)


@gpu
def test_policy_loss_is_deterministic_and_rows_are_independent():
    x, a, old, adv, ref = make((4097,), 200, "bf16", seed=11)
    o1, g1 = run_policy(x, a, old, adv, None, ref)
    o2, g2 = run_policy(x, a, old, adv, None, ref)
    assert torch.equal(o1.loss, o2.loss) and torch.equal(g1, g2)
    k = 1000
    w = torch.full((k,), 1.0 / 4097, device="cuda")
    o3, g3 = run_policy(x[:k], a[:k], old[:k], adv[:k], w, ref[:k])
    assert torch.equal(g3, g1[:k]) and torch.equal(o3.logp, o1.logp[:k])


@gpu
def test_policy_loss_large_offsets():
    """Rows whose elements start beyond 2^31 elements of the first."""
    V, rows = 40000, 3
    big = torch.empty((2 ** 31 + 5 * V,), dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((rows, V), (2 ** 30 + 7, 1))
    xs, a, old, adv, ref = make((rows,), V, "bf16", seed=12)
    x.copy_(xs)
    check_policy(x, a, old, adv, None, ref, name="offsets")


@gpu
def test_policy_loss_on_other_streams():
    x, a, old, adv, ref = make((512,), 1000, "bf16", seed=13)
    want, gw = run_policy(x, a, old, adv, None, ref)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(run_policy(x, a, old, adv, None, ref))
    torch.cuda.synchronize()
    for out, g in outs:
        assert torch.equal(out.loss, want.loss) and torch.equal(g, gw)


@gpu
@pytest.mark.parametrize("V,rows", [(14, 3000), (40, 3000), (3000, 64), (140003, 3)])
def test_policy_loss_in_a_graph(V, rows):
    """Forward and backward captured, replayed over new inputs between eager work."""
    from mobile_env.learning import policy_loss
    x, a, old, adv, ref = make((rows,), V, "bf16", seed=14)
    xs = x.detach().clone().requires_grad_()

    def step():
        out = policy_loss(xs, a, old, adv, ref_logp=ref, kl_coef=0.05, entropy_coef=0.01)
        g, = torch.autograd.grad(out.loss, xs)
        return out.loss.detach(), out.logp, g
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        nx = make((rows,), V, "bf16", seed=20 + k)
        with torch.no_grad():
            xs.copy_(nx[0])
        for dst, src in zip((a, old, adv, ref), nx[1:]):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want, gw = run_policy(nx[0], *nx[1:4], None, nx[4])
        assert torch.equal(got[0], want.loss.detach()) and torch.equal(got[1], want.logp)
        assert torch.equal(got[2], gw), k


@gpu
def test_policy_losses_in_two_graphs():
    """Two graphs with workspaces of their own, replayed in turn between eager calls."""
    from mobile_env.learning import policy_loss
    data = [make((4000,), V, "bf16", seed=60 + V) for V in (60, 140003 // 7)]
    data[1] = [t[:64].contiguous() if t is not None else None for t in data[1]]
    graphs, held = [], []
    for x, a, old, adv, ref in data:
        xs = x.requires_grad_()

        def step(xs=xs, a=a, old=old, adv=adv, ref=ref):
            out = policy_loss(xs, a, old, adv, ref_logp=ref, kl_coef=0.05, entropy_coef=0.01)
            return out.loss.detach(), torch.autograd.grad(out.loss, xs)[0]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(step())
        graphs.append(graph)
    for k in range(4):
        for x, a, old, adv, ref in data:
            adv.mul_(-1.25)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (x, a, old, adv, ref), (loss, g) in zip(data, held):
            want, gw = run_policy(x, a, old, adv, None, ref)
            assert torch.equal(loss, want.loss.detach()) and torch.equal(g, gw), k


@gpu
def test_policy_loss_as_a_node_of_autograd():
    """A freed graph, saved-tensor hooks, recomputed forward passes, hooks on the logits, several
    losses of one tensor, and what is refused."""
    from torch.utils.checkpoint import checkpoint
    from mobile_env.learning import policy_loss
    x, a, old, adv, ref = make((40,), 300, "f32", seed=18)
    _, want = run_policy(x, a, old, adv, None, ref)
    kw = dict(ref_logp=ref, kl_coef=0.05, entropy_coef=0.01)
    xs = x.clone().requires_grad_()
    loss = policy_loss(xs, a, old, adv, **kw).loss
    assert loss.grad_fn.name() == "PolicyLossBackward"
    loss.backward()
    assert torch.equal(xs.grad, want)
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()
    xs.grad = None
    seen = []
    xs.register_hook(lambda g: seen.append(g.clone()))
    with torch.autograd.graph.save_on_cpu():
        loss = policy_loss(xs, a, old, adv, **kw).loss
    (loss * 2).backward()
    check(xs.grad, want.double() * 2, 8 * U * want.double().abs(), "hooks", torch.float32)
    assert len(seen) == 1 and torch.equal(seen[0], xs.grad)
    y = x.clone().requires_grad_()
    checkpoint(lambda t: policy_loss(t * 1.0, a, old, adv, **kw).loss, y,
               use_reentrant=False).backward()
    assert torch.equal(y.grad, want)
    z = x.clone().requires_grad_()
    both = policy_loss(z, a, old, adv, **kw).loss + policy_loss(z, a, old, adv, **kw).loss
    both.backward()
    assert torch.equal(z.grad, want + want)
    out = policy_loss(z, a, old, adv, **kw)
    with pytest.raises(RuntimeError):
        out.logp.sum().backward()  # not differentiable
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(z, torch.ones_like(z))
        with pytest.raises(RuntimeError, match="forward-mode"):
            policy_loss(dual, a, old, adv)


@gpu
@pytest.mark.parametrize("V", [14, 300, 9000, 140003])
def test_policy_loss_backward_outside_its_forwards_graph(V):
    """Forward and backward in graphs of their own, the backward replayed alone over changing
    incoming gradients; then an eager backward, whose gradient a replay leaves as it is."""
    from mobile_env.learning import policy_loss
    x, a, old, adv, ref = make((9,), V, "bf16", seed=17)
    want, tol = policy64(x.cpu(), a.cpu(), old.cpu(), adv.cpu(), None, ref.cpu(), kl=0.05, ent=0.01)
    xs = x.clone().requires_grad_()
    incoming = torch.ones((), device="cuda")

    def forward():
        return policy_loss(xs, a, old, adv, ref_logp=ref, kl_coef=0.05, entropy_coef=0.01).loss
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(forward(), xs, incoming)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, stream=side):
        loss = forward()
    with torch.cuda.graph(second, stream=side, pool=first.pool()):
        g, = torch.autograd.grad(loss, xs, incoming, retain_graph=True)
    first.replay()
    for k, scale in enumerate((1.0, 2.0, 1.0, 0.5, 1.0)):
        incoming.fill_(scale)
        second.replay()
        torch.cuda.synchronize()
        check(g, want[3] * scale, tol[3] * scale, f"replay {k}", xs.dtype)
        g.zero_()  # (as a caller may that clips it in place)
    e, = torch.autograd.grad(loss, xs)
    torch.cuda.synchronize()
    check(e, want[3], tol[3], "eager", xs.dtype)
    keep = e.clone()
    with torch.no_grad():
        xs.mul_(0.5)
    first.replay()
    torch.cuda.synchronize()
    assert torch.equal(e, keep)


# -- advantages -----------------------------------------------------------------------------------
def adv64(r, d, v, last, gamma, lam, boot=True):
    r, v, last = (t.double().cpu().numpy() for t in (r, v, last))
    d = d.cpu().numpy().astype(bool)
    adv, tol = np.zeros_like(r), np.zeros_like(r)
    run, err, nxt = np.zeros_like(last), np.zeros_like(last), last
    for t in range(r.shape[0] - 1, -1, -1):
        cut = d[t] if r.ndim == 2 else d[t][:, None]
        b = gamma * nxt if boot else np.where(cut, 0.0, gamma * nxt)
        delta = r[t] + b - v[t]
        carried = np.where(cut, 0.0, gamma * lam * run)
        # four roundings of numbers no larger than their parts, doubled where a step is composed
        # with others before its turn; earlier errors shrink by gamma lam
        size = np.abs(r[t]) + np.abs(b) + np.abs(v[t]) + np.abs(carried)
        err = 8 * U * size + np.where(cut, 0.0, gamma * lam * err)
        run = delta + carried
        adv[t], tol[t], nxt = run, err, v[t]
    return adv, adv + v, tol, tol + 2 * U * np.abs(adv + v)


def check_adv(r, d, v, last, gamma=0.99, lam=0.95, boot=True, name=""):
    from mobile_env.learning import advantages
    a, ret = advantages(r, d, v, last, gamma, lam, bootstrap_done=boot)
    assert a.shape == r.shape and a.dtype == torch.float32 and a.is_contiguous()
    # the kernel's gamma and lam are float32; so are the oracle's
    g32, l32 = float(np.float32(gamma)), float(np.float32(lam))
    wa, wr, ta, tr = adv64(r, d, v, last, g32, l32, boot)
    check(a, torch.from_numpy(wa), torch.from_numpy(ta), name + " advantage")
    check(ret, torch.from_numpy(wr), torch.from_numpy(tr), name + " returns")


def make_adv(shape, dtype="f32", seed=0, p=0.07):
    g = torch.Generator().manual_seed(seed + 13 * len(shape) + shape[0])
    r = torch.randn(shape, generator=g)
    d = (torch.rand(shape[:2], generator=g) < p).to(torch.uint8)
    v = torch.randn(shape, generator=g).to(DT[dtype])
    last = torch.randn(shape[1:], generator=g).to(DT[dtype])
    return [t.cuda() for t in (r, d, v, last)]


@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [
    (1, 1), (2, 1), (1, 300), (20, 1), (20, 7), (20, 255), (20, 4097), (33, 64), (7, 17), (64, 3),
    (100, 5), (255, 2), (256, 16), (257, 9), (1000, 1), (2049, 1), (5000, 4), (8193, 1),
    # every pair of columns and lanes, whole and in segments, at their limits
    (400, 100), (512, 65), (513, 64), (700, 49), (2048, 5), (2049, 4), (3000, 100), (3000, 20),
    (128, 300), (129, 256), (32, 256), (33, 257), (1500, 260), (40, 9000), (8, 300), (9, 300),
    (20, 5, 30), (3, 1, 1), (20, 300, 15), (70, 2, 5), (513, 1, 7), (20, 0), (0, 4), (5, 3, 0)])
def test_advantages_shapes(shape, dtype):
    r, d, v, last = make_adv(shape, dtype)
    if 0 in shape:
        from mobile_env.learning import advantages
        a, ret = advantages(r, d, v, last)
        assert a.shape == ret.shape == shape
        return
    check_adv(r, d, v, last, name=str(shape))


@gpu
@pytest.mark.parametrize("boot", [True, False])
@pytest.mark.parametrize("gamma,lam", [(1.0, 1.0), (0.0, 0.5), (0.9, 0.0), (0.99, 0.95)])
@pytest.mark.parametrize("shape", [(40, 130), (300, 2), (20, 70000)])
def test_advantages_coefficients_and_ends(gamma, lam, boot, shape):
    r, d, v, last = make_adv(shape, seed=3)
    check_adv(r, d, v, last, gamma, lam, boot)
    d.fill_(1)
    check_adv(r, d, v, last, gamma, lam, boot, "every step done")
    d.zero_()
    check_adv(r, d.bool(), v, last, gamma, lam, boot, "no step done")


@gpu
def test_advantages_strides():
    """The multi-agent reward is column 3 of the observations; other orders and gaps."""
    from mobile_env.learning import advantages
    r, d, v, last = make_adv((23, 11, 6), seed=4)
    want = advantages(r, d, v, last)
    obs = torch.full((23, 11, 6, 4), float("nan"), device="cuda")
    obs[..., 3] = r
    vs = torch.full((6, 23, 22), float("nan"), device="cuda")
    vs[:, :, ::2] = v.permute(2, 0, 1)
    vs = vs[:, :, ::2].permute(1, 2, 0)
    ds = torch.full((11, 46), 7, dtype=torch.uint8, device="cuda")
    ds[:, ::2] = d.t()
    ds = ds[:, ::2].t()
    ls = last.t().contiguous().t()
    for got in (advantages(obs[..., 3], d, v, last), advantages(r, ds, vs, ls),
                advantages(r.flip(0).flip(0), d, v, last)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a reward and a value shared by all envs
    one = advantages(r[:, :1].expand(23, 11, 6), d, v[:, :1].expand(23, 11, 6), last)
    two = advantages(r[:, :1].repeat(1, 11, 1), d, v[:, :1].repeat(1, 11, 1), last)
    assert torch.equal(one[0], two[0])


@gpu
def test_advantages_nonfinite_values_stay_in_their_column_and_episode():
    from mobile_env.learning import advantages
    r, d, v, last = make_adv((50, 9), seed=5, p=0.0)
    d[30] = 1
    want = advantages(r, d, v, last)
    r[40, 2] = float("nan")
    v[35, 3] = float("inf")
    got = advantages(r, d, v, last)
    keep = torch.ones(50, 9, dtype=torch.bool)
    keep[31:41, 2] = False  # the done of step 30 stops it
    keep[31:36, 3] = False
    assert torch.isnan(got[0][40, 2]) and torch.isnan(got[0][31, 2])
    assert torch.equal(got[0][keep], want[0][keep])


@gpu
def test_advantages_of_a_rollout():
    """Straight from the engine's buffers, both reward forms, against the oracle."""
    import mobile_env
    env = mobile_env.make("mobile-large-ma-v0", num_envs=70, seed=5)
    env.reset()
    tr = env.engine.rollout(45)
    torch.cuda.synchronize()
    g = torch.Generator().manual_seed(1)
    v = torch.randn(45, 70, 30, generator=g).cuda()
    last = torch.randn(70, 30, generator=g).cuda()
    assert int(tr.done.sum()) == 2 * 70
    check_adv(tr.obs[..., 3], tr.done, v, last, name="ma")
    check_adv(tr.reward, tr.done, v[..., 0], last[..., 0], name="central")
    env.close()


@gpu
def test_advantages_in_a_graph():
    from mobile_env.learning import advantages
    r, d, v, last = make_adv((300, 40), seed=6)
    advantages(r, d, v, last)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = advantages(r, d, v, last)
    for k in range(3):
        for dst, src in zip((r, d, v, last), make_adv((300, 40), seed=30 + k)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = advantages(r, d, v, last)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# -- clip_grad_norm -------------------------------------------------------------------------------
def make_grads(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + len(sizes))
    return [(torch.randn(n, generator=g) * scale).to(DT[t]).cuda()
            for n, t in zip(sizes, dtypes)]


def check_clip(grads, max_norm, out=None, name=""):
    from mobile_env.learning import clip_grad_norm
    before = [g.clone() for g in grads]
    ref = math.sqrt(sum(float((g.double() ** 2).sum()) for g in before))
    norm = clip_grad_norm(grads, max_norm, out=out)
    # one rounding to float32 of a 64-bit sum (a level of its own error each)
    check(norm, torch.tensor(ref, dtype=torch.float64), U * ref * 1.001, name + " norm")
    f = max_norm / ref if ref > max_norm and math.isfinite(ref) else 1.0
    for g, b in zip(out if out is not None else grads, before):
        # the factor's rounding and the product's, then the type's
        want = b.double().cpu() * f
        check(g, want, 2.01 * U * want.abs() if f != 1.0 else 0.0, name + " gradient",
              b.dtype if f != 1.0 else None)
    if out is not None:
        for g, b in zip(grads, before):
            assert torch.equal(g, b)
    return norm


@gpu
@pytest.mark.parametrize("place", ["in", "out"])
@pytest.mark.parametrize("sizes", [
    [1], [0, 1, 0], [7, 8, 9], [2048, 2049, 2047], [120 * 256, 256, 256 * 256, 256, 256 * 14, 14],
    [100003, 5, 33333, 1], [3000001], [13] * 300, [1, 4097] * 130])
def test_clip_sizes(sizes, place):
    for k, dts in enumerate((["f32"], ["bf16"], ["f16"], ["f32", "bf16", "f16"])):
        grads = make_grads(sizes, (dts * len(sizes))[:len(sizes)], seed=k)
        out = [torch.full_like(g, float("nan")) for g in grads] if place == "out" else None
        check_clip(grads, 0.5, out, f"{sizes[:3]} {dts}")


@gpu
def test_clip_leaves_small_norms_and_nonfinite_ones():
    from mobile_env.learning import clip_grad_norm
    grads = make_grads([1000, 77], ["f32", "bf16"], seed=1, scale=1e-4)
    check_clip(grads, 1.0)                      # below: bits unchanged
    check_clip([torch.zeros(5, device="cuda")], 0.0)   # 0 is not above 0
    check_clip([torch.zeros(0, device="cuda")], 1.0, name="nothing at all")
    check_clip(make_grads([50], ["f32"]), 0.0, name="to nothing")
    for bad in (float("inf"), float("nan")):
        g = make_grads([1000, 77], ["f32", "bf16"], seed=2)
        g[1][3] = bad
        keep = [t.clone() for t in g]
        out = [torch.empty_like(t) for t in g]
        norm = clip_grad_norm(g, 0.5, out=out)
        assert not math.isfinite(float(norm))
        norm = clip_grad_norm(g, 0.5)
        assert not math.isfinite(float(norm))
        for a, b, c in zip(g, keep, out):
            same = (a == b) | (torch.isnan(a) & torch.isnan(b))
            assert same.all() and ((c == b) | (torch.isnan(c) & torch.isnan(b))).all()


@gpu
def test_clip_values_whose_squares_leave_float32():
    check_clip([torch.full((1000,), 1e30, device="cuda")], 1.0, name="large")
    check_clip([torch.full((1000,), 1e-30, device="cuda")], 1e-29, name="tiny")
    from mobile_env.learning import clip_grad_norm
    g = torch.full((1000,), 3e38, device="cuda")  # a norm beyond float32 is not finite
    assert float(clip_grad_norm([g], 1.0)) == math.inf and (g == 3e38).all()


@gpu
def test_clip_views_and_orders():
    """Offset views, other axis orders, and nothing written beside them."""
    buf = torch.randn(4000, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    keep = buf.clone()
    a, b = buf[3:1004], buf[1005:2005].view(10, 100).t()
    check_clip([a, b], 0.5)
    from mobile_env.learning import clip_grad_norm
    one = torch.arange(6.0, device="cuda").view(2, 3)  # a tensor is a list of itself
    assert abs(float(clip_grad_norm(one, 1.0)) - math.sqrt(55.0)) <= 8 * U
    assert abs(float(one.double().norm()) - 1.0) <= 4 * U
    for s in (slice(0, 3), slice(1004, 1005), slice(2005, 4000)):
        assert torch.equal(buf[s], keep[s])


@gpu
def test_clip_refuses_shared_memory():
    from mobile_env.learning import clip_grad_norm
    g = torch.randn(100, device="cuda")
    keep = g.clone()
    for bad in ([g, g], [g[:60], g[50:]]):
        with pytest.raises(ValueError):
            clip_grad_norm(bad, 1.0)
    with pytest.raises(ValueError):
        clip_grad_norm([g[:50]], 1.0, out=[g[10:60]])
    assert torch.equal(g, keep)


@gpu
def test_clip_counts_as_a_write():
    """Autograd sees that a clipped tensor changed."""
    from mobile_env.learning import clip_grad_norm
    g = torch.randn(10, device="cuda")
    p = torch.ones(10, device="cuda", requires_grad=True)
    y = (p * g).sum()
    clip_grad_norm([g], 0.1)
    with pytest.raises(RuntimeError):
        y.backward()


@gpu
def test_clip_in_graphs():
    """Two captured graphs replayed in turn with eager calls between share nothing."""
    from mobile_env.learning import clip_grad_norm
    sets = [make_grads([5000, 17, 300], ["f32", "bf16", "f16"], seed=40 + k) for k in range(2)]
    outs = [[torch.empty_like(t) for t in s] for s in sets]
    clip_grad_norm(sets[0], 0.5, out=outs[0])
    torch.cuda.synchronize()
    graphs, norms = [], []
    for s, o in zip(sets, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(clip_grad_norm(s, 0.5, out=o))
        graphs.append(graph)
    for k in range(4):
        for s in sets:
            for t in s:
                t.mul_(1.5)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s, o, n in zip(sets, outs, norms):
            want = [torch.empty_like(t) for t in s]
            wn = clip_grad_norm(s, 0.5, out=want)
            assert torch.equal(n, wn) and all(torch.equal(x, y) for x, y in zip(o, want))
