"""How the policy operators (mobile_env.learning) launch their work, as far as the host decides it:
workspaces, launches, limits."""
import ctypes as C

import pytest
import torch

from mobile_env.core import _native as N

gpu = pytest.mark.gpu


def _adv_workspace(T, E, U=1):
    a = N.MevAdvantages(T=T, E=E, U=U)
    return N.lib().mev_advantages_workspace(C.byref(a))


# steps and columns that 256 lanes of 8 steps hold at once: 4 lanes a column from 256 columns on, 16
# from 64, 64 from 4, all of them below; two tiles of one lane a column where columns abound
@pytest.mark.parametrize("T,E", [
    (1, 1), (8, 1000), (9, 1000), (10, 1000), (16, 1000), (32, 1000), (9, 256), (16, 256),
    (16, 32768), (16, 65536), (10, 100000), (10, 131072), (16, 262144), (9, 300), (33, 64), (40, 100),
    (64, 100), (128, 64), (33, 4), (64, 5), (129, 63), (200, 3), (512, 4), (33, 1), (64, 1),
    (129, 1), (600, 3), (1024, 1), (1025, 1), (2048, 1)])
def test_a_rollout_of_one_tile_is_one_launch(T, E):
    """A workspace is asked only where a rollout is cut into segments."""
    assert _adv_workspace(T, E) == 0


def test_long_rollouts_of_few_columns_are_cut():
    for T, E in ((2049, 1), (5000, 4), (20000, 800)):
        assert _adv_workspace(T, E) > 0


# tiles of 2,048 steps of one column, of 512 of four
@pytest.mark.parametrize("T,E,segments", [(2049, 1, 2), (4096, 1, 2), (4097, 1, 3), (5000, 4, 10)])
def test_traces_are_formed_of_what_lies_behind_a_segment(T, E, segments):
    """Two floats a column for each segment but the one of the first steps, which none needs."""
    assert _adv_workspace(T, E) == 8 * E * (segments - 1)


@gpu
@pytest.mark.parametrize("T,E", [(2049, 1), (4097, 1), (5000, 4), (20000, 70), (2049, 300)])
def test_advantages_in_segments(T, E):
    from test_learning import check_adv, make_adv
    check_adv(*make_adv((T, E), seed=E), name=f"{T} x {E}")
    r, d, v, last = make_adv((T, E), seed=E, p=0.0)
    check_adv(r, d, v, last, gamma=1.0, lam=1.0, name=f"{T} x {E}, one episode")


@gpu
@pytest.mark.parametrize("T,E", [(9, 1000), (16, 1000), (16, 65536), (10, 65537), (9, 300000),
                                 (33, 1), (64, 100), (129, 3), (600, 3), (1024, 1), (129, 63)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_advantages_of_one_tile(T, E, dtype):
    from test_learning import check_adv, make_adv
    r, d, v, last = make_adv((T, E), dtype, seed=T)
    check_adv(r, d, v, last, name=f"{T} x {E}")
    check_adv(r, d, v, last, boot=False, name=f"{T} x {E}, ends")


@gpu
def test_advantages_of_more_columns_than_one_axis_of_a_grid():
    """2^32 lanes and more, offsets beyond 32 bits: one step of 4.3 billion envs, whose rewards and
    done flags are shared (outputs 34 GB)."""
    from mobile_env.learning import advantages
    E = (1 << 32) + 301
    v = torch.empty((1, E), dtype=torch.bfloat16, device="cuda").normal_()
    r = torch.full((1, 1), 0.5, device="cuda").expand(1, E)
    d = torch.zeros((1, 1), dtype=torch.uint8, device="cuda").expand(1, E)
    last = torch.zeros(1, dtype=torch.bfloat16, device="cuda").expand(E)
    adv, ret = advantages(r, d, v, last)
    for a in range(0, E, 1 << 28):
        s = slice(a, min(E, a + (1 << 28)))
        want = 0.5 - v[0, s].float()
        assert torch.equal(adv[0, s], want), a
        assert torch.equal(ret[0, s], want + v[0, s].float()), a


def test_split_rows_beyond_a_grid_are_refused():
    """Rows of one shared row of logits, say: more workgroups than one launch takes."""
    fake = 1 << 20  # never read
    a = N.MevPolicy(logits=fake, action=fake, logp=fake, entropy=fake, workspace=fake,
                    workspace_bytes=1 << 62, rows=1 << 26, inner=1 << 26, actions=200000,
                    action_bytes=8)
    assert N.lib().mev_policy_rows(C.byref(a), None) == N.MEV_EINVAL


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[1003], [5, 4099, 0, 70001], [3_000_001] * 2])
def test_clip_by_a_factor_below_the_normal_numbers(sizes, dtype):
    """The factor 1e-12 / 1e31 and less; the products are ordinary numbers, off by the factor's
    rounding and the product's (a scale by 2^-100 is exact)."""
    from mobile_env.learning import clip_grad_norm
    from test_learning import DT, U, check
    g = torch.Generator().manual_seed(len(sizes))
    for max_norm in (1e-12, 1e-18):
        grads = [(torch.randn(n, generator=g) * 1e30).to(DT[dtype]).cuda() for n in sizes]
        norm = sum(float(t.double().square().sum()) for t in grads) ** 0.5
        want = [t.double().cpu() * (float(torch.tensor(max_norm)) / norm) for t in grads]
        clip_grad_norm(grads, max_norm)
        for t, w in zip(grads, want):
            check(t, w, 2.01 * U * w.abs(), f"{max_norm}", t.dtype)


# -- offsets beyond 32 bits ------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("V", [40000, 70001])
def test_gradients_beyond_32_bits(V):
    """2.8 billion logits and as many gradients; rows with weight at both ends alone."""
    from mobile_env.learning import policy_loss
    from test_learning import check, make, policy64
    rows = 2_800_000_000 // V
    x, a, old, adv, ref = make((6,), V, "bf16", seed=31, dev="cpu")
    want, tol = policy64(x, a, old, adv, None, ref, kl=0.05, ent=0.01)
    at = torch.tensor([0, 1, rows // 2, rows - 3, rows - 2, rows - 1])
    big = torch.full((rows, V), float("nan"), dtype=torch.bfloat16, device="cuda")
    big[at.cuda()] = x.cuda()

    def spread(t):
        out = torch.zeros(rows, dtype=t.dtype)
        out[at] = t
        return out.cuda()
    w = spread(torch.full((6,), 1 / 6))
    big.requires_grad_()
    out = policy_loss(big, spread(a), spread(old), spread(adv), weight=w, ref_logp=spread(ref),
                      kl_coef=0.05, entropy_coef=0.01)
    out.loss.backward()
    check(out.logp[at.cuda()], want[1], tol[1], "logp")
    check(out.loss, want[0], tol[0] + 2.0 ** -23 * want[0].abs(), "loss", torch.float32)
    g = big.grad
    # (six sixths of float32, off by half a step each)
    check(g[at.cuda()], want[3], tol[3] + 2.0 ** -23 * want[3].abs(), "gradient", torch.bfloat16)
    for s in range(0, rows, 8192):
        rest = g[s:s + 8192]
        keep = w[s:s + 8192] == 0
        assert not rest[keep].any(), s


@gpu
def test_clipping_beyond_32_bits():
    """One gradient of 4.4 billion elements."""
    from mobile_env.learning import clip_grad_norm
    n = (1 << 32) + 100_003
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    spots = torch.tensor([0, 1, (1 << 31) - 1, 1 << 31, (1 << 32) - 1, 1 << 32, n - 1]).cuda()
    g[spots] = torch.tensor([1.0, -2.0, 4.0, 8.0, -4.0, 2.0, 1.0], dtype=torch.bfloat16).cuda()
    want = g[spots].double()
    norm = clip_grad_norm(g, 0.5)
    total = (want ** 2).sum().sqrt()
    assert abs(float(norm) - float(total)) <= 2.0 ** -23 * float(total)
    # half a step of bf16, and of float32 for the factor and the product
    off = (g[spots].double() - want * 0.5 / total).abs() / (want * 0.5 / total).abs()
    assert float(off.max()) <= 2.0 ** -8 + 2.0 ** -22
    g[spots] = 0
    assert not g.any()
