"""Rows of the policy operators (mobile_env.learning) whose mass lies where a fault would: at a row's
end, where the kernels' last vector repeats elements of the one before; and long rows at the
tolerance of the sums that their lanes form."""
import math

import pytest
import torch

from test_learning import DT, U, check, make, policy64, rows64, run_policy

gpu = pytest.mark.gpu

# about as long as what a workgroup holds in its registers, and beyond it
LONG = [4099, 8193, 12289, 16391, 20481, 24581, 32769, 40961, 41567, 49153, 49159, 57345, 65543, 81923,
        98311, 114697, 131071, 131073, 140003, 200001]


def heavy(rows, V, dtype, seed=0):
    """Rows whose last 17 logits (the last vector, the one before, and one more) hold nearly all of
    the mass, the action among them; row 0 with its mass in the very last logit, row 1 in the one
    before the last vector of 8, row 2 in the first."""
    g = torch.Generator().manual_seed(1000 * seed + V)
    x = torch.randn(rows, V, generator=g)
    x[:, -17:] += 14.0
    x[0, -1] += 6.0
    x[1, -9] += 6.0
    x[2, 0] += 20.0
    x = x.to(DT[dtype])
    a = V - 1 - torch.randint(0, 17, (rows,), generator=g)
    a[2] = 0
    L = rows64(x, a)[0]
    old = (L - 0.05 - 0.05 * torch.rand(rows, generator=g).double()).float()
    adv = torch.randn(rows, generator=g)
    ref = (L + 0.2 * torch.randn(rows, generator=g).double()).float()
    return x, a, old, adv, ref


# -- the oracle, on the CPU: what the GPU tests below would see ------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", LONG)
def test_a_lost_or_doubled_element_is_beyond_the_tolerances(V, dtype):
    """Each of a row's last eight elements, counted twice or not at all, moves the log-probability or
    the entropy of some row by more than ten of its tolerances."""
    x, a, old, adv, ref = heavy(4, V, dtype)
    want, tol = policy64(x, a, old, adv, None, ref, kl=0.05, ent=0.01)
    d = x.double() - x.double().amax(-1, keepdim=True)
    s = d.exp().sum(-1)
    t = (d.exp() * d).sum(-1)
    da = d.gather(-1, a[:, None])[:, 0]
    for k in range(1, 9):
        e = d[:, -k].exp()
        for sign in (1.0, -1.0):
            s2, t2 = s + sign * e, t + sign * e * d[:, -k]
            off = torch.maximum((da - s2.log() - want[1]).abs() / tol[1],
                                (s2.log() - t2 / s2 - want[2]).abs() / tol[2])
            assert off.max() > 10, (k, sign, off)


# -- on the GPU ------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", LONG)
def test_rows_with_their_mass_at_the_end(V, dtype):
    """In few rows (where they are split over workgroups) and among many without weight (where one
    workgroup holds each that fits)."""
    from mobile_env.learning import action_logp
    x, a, old, adv, ref = heavy(4, V, dtype)
    want, tol = policy64(x, a, old, adv, None, ref, kl=0.05, ent=0.01)
    x, a, old, adv, ref = (t.cuda() for t in (x, a, old, adv, ref))
    out, g = run_policy(x, a, old, adv, None, ref)
    for name, got, k in (("logp", out.logp, 1), ("entropy", out.entropy, 2), ("loss", out.loss, 0)):
        check(got, want[k], tol[k], f"V={V} {name}")
    check(g, want[3], tol[3], f"V={V} gradient", x.dtype)
    logp, ent = action_logp(x, a)
    check(logp, want[1], tol[1], "action_logp logp")
    check(ent, want[2], tol[2], "action_logp entropy")
    rows = 164 if V > 65536 // (2 if dtype == "f32" else 1) else 4
    at = torch.tensor([0, 1, rows - 2, rows - 1], device="cuda")
    big = [torch.zeros((rows,) + t.shape[1:], dtype=t.dtype, device="cuda")
           for t in (x, a, old, adv, ref)]
    for b, t in zip(big, (x, a, old, adv, ref)):
        b[at] = t
    w = torch.zeros(rows, device="cuda")
    w[at] = 0.25
    out, g = run_policy(*big[:4], w, big[4])
    check(out.logp[at], want[1], tol[1], "logp among many")
    check(out.entropy[at], want[2], tol[2], "entropy among many")
    check(g[at], want[3], tol[3], "gradient among many", x.dtype)
    g[at] = 0
    assert not g.any()


def tight(x, a):
    """Log-probability, entropy and their tolerances, with the longest sum of any layout: 128 terms
    of a lane (16 vectors of 8) or 32 at a time and a join for each 32,768, 10 levels of lanes, and
    two roundings a join; a term is off by U |x - m| from its argument's rounding, which averages
    to D = H - ln s over the terms' weights (H = ln s - t / s, and t = sum e^(x-m) (x-m) <= 0), and
    by 4 U."""
    L, H, _, _ = rows64(x, a)
    xs = x.double()
    m = xs.amax(-1)
    lns = (xs - m[:, None]).exp().sum(-1).log()
    D = H - lns
    rel = U * (8 + 4 * D + 160)
    xa = xs.gather(-1, a[:, None])[:, 0] - m
    return L, H, rel + 4 * U * (xa.abs() + lns), rel * (1 + 2 * D) + 4 * U * (lns + D)


@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", LONG + [300001])
def test_long_rows_at_the_tolerance_of_their_sums(V, dtype):
    from mobile_env.learning import action_logp
    for rows in (3, 161):
        if rows * V > 6_600_000:
            continue
        x, a, *_ = make((rows,), V, dtype, seed=rows, spread=3.0, dev="cpu")
        L, H, tl, th = tight(x, a)
        logp, ent = action_logp(x.cuda(), a.cuda())
        check(logp, L, tl, f"{rows} x {V} logp", torch.float32)
        check(ent, H, th, f"{rows} x {V} entropy", torch.float32)


@gpu
@pytest.mark.parametrize("V", [5, 13, 30, 300, 9000, 140003])
@pytest.mark.parametrize("dtype", list(DT))
def test_ratios_beyond_float32(V, dtype):
    """Where the advantage is 0, so are the loss and the gradient, as they are with a ratio that
    float32 holds; other rows of the batch keep theirs."""
    x, a, old, *_ = make((6,), V, dtype, seed=21, dev="cpu")
    L = rows64(x, a)[0]
    old = (L - torch.tensor([100.0, 89.0, -300.0, 95.0, 180.0, 0.1], dtype=torch.float64)).float()
    adv = torch.tensor([0.0, 0.0, -1.0, 0.0, 0.0, 1.0])
    w = torch.full((6,), 0.25)
    want, tol = policy64(x, a, old, adv, w, None, ent=0.01)
    assert want[3].isfinite().all() and want[3].abs().max() > 0.01
    out, g = run_policy(x.cuda(), a.cuda(), old.cuda(), adv.cuda(), w.cuda(), None, ent=0.01)
    check(g, want[3], tol[3], "gradient", x.dtype)
    check(out.loss, want[0], tol[0], "loss", torch.float32)
    # a behaviour policy that could not have taken the action: the loss says so
    old[0] = -math.inf
    out, g = run_policy(x.cuda(), a.cuda(), old.cuda(), adv.cuda(), w.cuda(), None, ent=0.01)
    assert torch.isnan(out.loss)


@gpu
@pytest.mark.parametrize("V", [11, 40, 300, 3001, 140003])
def test_small_probabilities_keep_their_digits(V):
    """The gradient's entries relative to themselves, f32, where the gradient is the probability
    (ratio, advantage and weight 1) and the differences x - m are exact: p = e^(x - m) / s.
    x - m lies in (-22, -11.1], its product with log2 e in (-32, -16] is rounded by half a step of
    2^-19 (times ln 2: 6.7e-7), the constant log2 e by 1.4e-8 of it (3e-7 of p at most); e^x and 1 / s
    are good to a step (1.2e-7 each), s itself to 8 of its half steps (it is 1 and V / 10^5 at most),
    and two products are rounded: 1.81e-6 with 10 U for those and the coefficient."""
    from mobile_env.learning import action_logp, policy_loss
    rows = 24 if V < 100000 else 3
    g = torch.Generator().manual_seed(V)
    x = -torch.randint(2850, 5600, (rows, V), generator=g).float() / 256
    x[:, 0] = 0.0
    x = x.cuda()
    a = torch.zeros(rows, dtype=torch.int64, device="cuda")
    old, _ = action_logp(x, a)
    p = x.clone().requires_grad_()
    out = policy_loss(p, a, old, torch.ones(rows, device="cuda"), torch.ones(rows, device="cuda"))
    grad, = torch.autograd.grad(out.loss, p)
    want = torch.softmax(x.cpu().double(), -1)[:, 1:]
    off = ((grad[:, 1:].cpu().double() - want) / want).abs().max().item()
    assert off <= 6.7e-7 + 3e-7 + 2 * 2.0 ** -23 + 10 * U, off
