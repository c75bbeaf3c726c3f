"""Policy losses at the ends of what the header allows: reference policies without any probability, logits of -inf where
something is asked of them, very large logits, targets of any scale."""
import math

import numpy as np
import pytest

from test_policy_loss_gpu import TYPES, dtype_of, half_step, pack, ref_clipped, ref_search, relative_bound

pytestmark = pytest.mark.gpu

LENGTHS = [7, 225, 1000, 4672, 40000, 300007]        # lanes, warps, CTAs, clusters, clusters over device memory
INF = float("inf")


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


def floor_of(dt):
    """What a difference of logits of -inf counts as."""
    return -1.5703125 * 2.0 ** 99 if dt == "bf16" else -1e30


def cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("many", [1, 500], ids=["few", "many"])
@pytest.mark.parametrize("A", LENGTHS)
@pytest.mark.parametrize("dt", TYPES)
def test_reference_without_any_probability(api, dt, A, many):
    """KL(p | q) is +infinity where q gives no legal action any probability: so is the loss, whose gradient is that of its
    other terms; without a KL term the loss is what it is without a reference.  Rows between such rows are as ever."""
    import torch
    n = 6 * (many if A <= 1000 else 1 + many // 100)
    T = dtype_of(dt)
    rng = np.random.default_rng(A)
    z = torch.from_numpy(rng.normal(0, 2, (n, A)).astype(np.float32)).to(T)
    zr = torch.from_numpy(rng.normal(0, 2, (n, A)).astype(np.float32)).to(T)
    legal = rng.random((n, A)) < 0.7
    legal[:, A // 2] = True
    legal[3::6] = False
    legal[3::6, A // 2] = True
    zr64 = zr.double().numpy()
    none = np.zeros(n, bool)
    none[1::3] = none[3::6] = True
    zr[torch.from_numpy(none[:, None] & legal)] = -INF
    act = np.full(n, A // 2, np.int32)
    z64 = z.double().numpy()
    w, adv = rng.uniform(0.5, 2, n).astype(np.float32), rng.normal(0, 1, n).astype(np.float32)
    old = np.full(n, -3.0, np.float32)
    args = (cuda(act), cuda(old), cuda(adv), pack(legal))
    half, least = half_step(T)
    reach = 2 * max(np.abs(z64).max(), np.abs(zr64).max()) + 1
    D = relative_bound(A, reach)
    E = 4 * D * (1 + reach)
    for kappa in (0.3, 0.0):
        loss, grad, stats = [x.double().cpu().numpy() for x in
                             api.policy_loss_clipped(z.cuda(), *args, zr.cuda(), cuda(w), kl_coef=kappa, entropy_coef=0.05)]
        assert (stats[none, 2] == INF).all()
        if kappa:
            assert (loss[none] == INF).all()
        for rows, k, ref in ((none, 0.0, None), (~none, kappa, zr64)):
            rl, rg, rs, terms, lterm = ref_clipped(z64[rows], legal[rows], act[rows], old[rows].astype(float), adv[rows].astype(float),
                                                   None if ref is None else ref[rows], w[rows].astype(float), 0.2, 0.2, k, 0.05)
            assert (np.abs(grad[rows] - rg) <= (4 * D + reach * 2.0 ** -22) * (terms + np.abs(rg)) + half * np.abs(rg) + least).all()
            keep = [0, 1, 3] if ref is None else [0, 1, 2, 3]
            assert (np.abs(stats[rows] - rs)[:, keep] <= (E * (1 + np.abs(rs)))[:, keep]).all()
            if k == kappa or not kappa:
                assert (np.abs(loss[rows] - rl) <= E * (np.abs(rl) + lterm + w[rows])).all()


@pytest.mark.parametrize("unlike", [False, True], ids=["alike", "unlike"])
@pytest.mark.parametrize("A", LENGTHS)
@pytest.mark.parametrize("dt", TYPES)
def test_targets_at_logits_of_minus_infinity(api, dt, A, unlike):
    """A legal logit of -inf that the target wants, in the same measure whatever the type and the length; rows that want none
    of theirs are as if those were not legal."""
    import torch
    n = 40
    T = dtype_of(dt)
    rng = np.random.default_rng(A + 1)
    z = torch.from_numpy(rng.normal(0, 2, (n, A)).astype(np.float32)).to(T)
    t = rng.gamma(1.0, 1.0, (n, A)).astype(np.float32)
    gone = rng.random((n, A)) < 0.2
    gone[:, 0] = False
    gone[::2, A - 1] = gone[1::4, A // 2] = True
    z64 = z.double().numpy()
    t[gone] = 0
    wanted = np.arange(n) % 2 == 0
    share = np.float32(0.01)
    t[wanted, A - 1] = t[wanted].sum(1) * share / (1 - share)
    zc = z.clone()
    zc[torch.from_numpy(gone)] = -INF
    zd = zc.cuda()
    if unlike:
        zd = torch.nn.functional.pad(zd, (0, 3))[:, :A]
    loss, grad, stats = [x.double().cpu().numpy() for x in api.policy_loss_search(zd, cuda(t), entropy_coef=0.05)]
    rl, rg, rs, terms = ref_search(z64, ~gone, np.where(gone, 0, t).astype(float), np.ones(n), 0.05)
    # the reference above knows nothing of what is gone: its pi is of the rest
    t64 = t.astype(float)
    pi_all = t64 / t64.sum(1, keepdims=True)
    want_g = rg + np.where(gone, 0, t64) / np.where(gone, 0, t64).sum(1, keepdims=True) - pi_all
    reach = 2 * np.abs(z64).max() + 1
    D = relative_bound(A, reach)
    half, least = half_step(T)
    assert (np.abs(grad - want_g) <= 4 * D * (terms + pi_all) + half * np.abs(want_g) + least).all()
    missing = np.where(gone, pi_all, 0).sum(1)
    ce = rs[:, 0] * (1 - missing) + missing * -floor_of(dt)
    # a rounding for each of the products and sums of 1e30, besides those of the ordinary ones
    assert (np.abs(stats[:, 0] - ce) <= 4 * D * (1 + reach + ce)).all()
    assert (np.abs(stats[:, 1] - rs[:, 1]) <= 4 * D * (1 + reach + rs[:, 1])).all()
    assert (np.abs(loss - (ce - 0.05 * rs[:, 1])) <= 4 * D * (1 + reach + ce) * 1.05).all()


@pytest.mark.parametrize("A", LENGTHS)
@pytest.mark.parametrize("dt", TYPES)
def test_actions_the_reference_excludes(api, dt, A):
    """KL counts an action that q excludes as -1e30, whatever the type and the length; an action whose own logit is -inf has
    the ratio 0 and no gradient."""
    import torch
    n = 24
    T = dtype_of(dt)
    rng = np.random.default_rng(A + 2)
    z = torch.from_numpy(rng.normal(0, 2, (n, A)).astype(np.float32)).to(T)
    zr = torch.from_numpy(rng.normal(0, 2, (n, A)).astype(np.float32)).to(T)
    at = A // 3
    zr[::3, at] = -INF                           # excluded by q
    z[1::3, at] = zr[1::3, at] = -INF            # by both: nothing to count
    act = np.full(n, at, np.int32)
    act[::3] = 0
    z64, r64 = z.double().numpy(), zr.double().numpy()
    legal = np.ones((n, A), bool)
    legal[1::3, at] = False                      # for the reference result: p is 0 there
    low = floor_of(dt)
    logp = z64 - np.where(legal, z64, -INF).max(1, keepdims=True)
    d = np.where(legal, logp, low)
    e = np.where(legal, np.exp(d), 0)
    p = e / e.sum(1, keepdims=True)
    lp = np.where(legal, d - np.log(e.sum(1, keepdims=True)), 0)
    dr = r64 - np.where(np.isfinite(r64), r64, -INF).max(1, keepdims=True)
    dr = np.where(np.isfinite(dr), dr, low)
    x = np.where(legal, lp - (dr - np.log(np.exp(dr).sum(1, keepdims=True))), 0)
    kl = (p * x).sum(1)
    kappa, w = 0.25, rng.uniform(0.5, 2, n).astype(np.float32)
    loss, grad, stats = api.policy_loss_clipped(z.cuda(), cuda(act), cuda(np.zeros(n, np.float32)), cuda(np.zeros(n, np.float32)), None, zr.cuda(),
                                                cuda(w), kl_coef=kappa)
    loss, stats = loss.double().cpu().numpy(), stats.double().cpu().numpy()
    reach = 2 * max(np.abs(z64[legal]).max(), np.abs(r64[np.isfinite(r64)]).max()) + 1
    D = relative_bound(A, reach)
    size = (p * np.abs(x)).sum(1)
    assert (np.abs(stats[:, 2] - kl) <= 4 * D * (1 + reach + size)).all()
    assert (np.abs(loss - w * kappa * kl) <= 4 * D * w * (1 + reach + size)).all()
    gone = np.arange(n) % 3 == 1
    assert (stats[gone, 1] == 0).all() and (np.abs(stats[gone, 0] / low - 1) <= 2.0 ** -20).all()
    # in fp32: what is beyond the gradient's type becomes infinite in it
    want = w[:, None] * kappa * p * (x - kl[:, None])
    tol = 4 * D * w[:, None] * kappa * p * (np.abs(x) + size[:, None] + 1)
    top = float(torch.finfo(T).max)
    got = grad.double().cpu().numpy()
    half, least = half_step(T)
    big = np.abs(want) > top
    sure = np.abs(want) - tol > top * (1 + half)
    assert (got[sure] == np.sign(want[sure]) * INF).all()
    fine = ~big & (np.abs(want) + tol < top)
    assert (np.abs(got - want)[fine] <= (tol + half * np.abs(want) + least)[fine]).all()
    assert (got[gone, at] == 0).all()


@pytest.mark.parametrize("A", LENGTHS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("total", [1e-37, 1e-30, 1e-15, 1e7, 1e9, 1e20, 1e30, 8e37])
def test_targets_of_any_scale(api, dt, A, total):
    """Loss and gradient do not depend on the scale of the targets, with logits far apart and the weight of a loss scale."""
    import torch
    n = 10
    T = dtype_of(dt)
    rng = np.random.default_rng(A + 3)
    z = torch.from_numpy(rng.normal(0, 8, (n, A)).astype(np.float32)).to(T)
    t = rng.gamma(0.5, 1.0, (n, A))
    t = (t / t.sum(1, keepdims=True) * total).astype(np.float32)
    t[3] = 0
    legal = rng.random((n, A)) < 0.8
    legal[:, 1] = True
    w = np.full(n, 1024.0, np.float32)
    z64 = z.double().numpy()
    loss, grad, stats = [x.double().cpu().numpy() for x in api.policy_loss_search(z.cuda(), cuda(t), pack(legal), cuda(w), entropy_coef=0.05)]
    rl, rg, rs, terms = ref_search(z64, legal, t.astype(float), w.astype(float), 0.05)
    reach = 2 * np.abs(z64).max() + 1
    D = relative_bound(A, reach)
    half, least = half_step(T)
    top = float(torch.finfo(T).max)
    assert np.abs(rg).max() < top
    assert (np.abs(grad - rg) <= 4 * D * terms + half * np.abs(rg) + least).all()
    assert (np.abs(stats - rs) <= 4 * D * np.stack([1 + reach + rs[:, 0], 1 + reach + rs[:, 1], rs[:, 2], 1 + reach + np.abs(rs[:, 3])], 1)).all()
    assert (np.abs(loss - rl) <= 4 * D * (np.abs(rl) + w * 1.05 * (1 + reach))).all()


@pytest.mark.parametrize("A", LENGTHS)
def test_visit_counts_beyond_32_bits_in_sum(api, A):
    """The largest counts, some of them at logits of -inf: 6e9 visits of which a third are at -1e30."""
    import torch
    z = np.zeros((3, A), np.float32)
    z[:, 5] = -INF
    z[1] = -INF
    z[1, 2] = 0
    t = np.zeros((3, A), np.int32)
    t[0, [2, 4, 5]] = t[1, [2, 4, 5]] = 2000000000
    t[2, 2] = 2147483647
    loss, grad, stats = [x.double().cpu().numpy() for x in api.policy_loss_search(cuda(z), cuda(t))]
    D = relative_bound(A, 1)
    assert abs(stats[0, 0] - 1e30 / 3) <= 4 * D * 1e30 and abs(stats[1, 0] - 2e30 / 3) <= 4 * D * 1e30
    assert abs(stats[2, 0] - math.log(A - 1)) <= 4 * D * (1 + math.log(A))
    assert np.allclose(stats[:, 2], [6e9, 6e9, 2147483647.0], rtol=2.0 ** -22) and np.isfinite(loss).all()
    assert abs(grad[1, 4] + 1 / 3) <= 4 * D and abs(grad[1, 2] - 2 / 3) <= 4 * D and abs(grad[0, 5] + 1 / 3) <= 4 * D


@pytest.mark.parametrize("A", LENGTHS)
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_very_large_logits(api, dt, A):
    """One logit of 1e36 among ordinary ones: the policy is that action, the others count as -1e30."""
    import torch
    T = dtype_of(dt)
    z = torch.zeros((2, A), dtype=T)
    z[:, 3] = 1e36
    z[1] *= -1                                   # one logit of -1e36 among zeros
    t = np.full((2, A), 800, np.int32)
    loss, grad, stats = [x.double().cpu().numpy() for x in api.policy_loss_search(z.cuda(), cuda(t), entropy_coef=0.05)]
    D, low = relative_bound(A, 1), floor_of(dt)
    half = half_step(T)[0]
    ce = np.array([(A - 1) / A * -low, -low / A])
    # of the second row's, in the order of 1e30, the logarithm is lost
    assert (np.abs(stats[:, 0] - ce) <= (4 * D + 2.0 ** -20) * ce).all()
    assert stats[0, 1] == 0 and abs(stats[1, 1] - math.log(A - 1)) <= 4 * D * (1 + math.log(A))
    assert abs(grad[0, 3] - (A - 1) / A) <= 4 * D + half and (np.abs(grad[0, 4:] + 1 / A) <= (4 * D + half) / A).all()
    assert abs(grad[1, 3] + 1 / A) <= (4 * D + half) / A


@pytest.mark.parametrize("where", ["logits", "reference"])
@pytest.mark.parametrize("A", LENGTHS)
@pytest.mark.parametrize("dt", TYPES)
def test_plus_infinity_makes_its_row_nan(api, dt, A, where):
    """A legal +inf, of the logits or the reference, makes loss, gradient and the statistics that depend on it NaN; at an
    action that is not legal it does not matter."""
    import torch
    n, T = 9, dtype_of(dt)
    g = torch.Generator(device="cuda")
    g.manual_seed(A)
    z, zr = torch.randn((2, n, A), generator=g, device="cuda").to(T)
    x = z if where == "logits" else zr
    x[::3, A // 2] = INF
    x[1::3, A - 1] = INF
    legal = np.ones((n, A), bool)
    legal[1::3, A - 1] = False
    act, one = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.ones(n, device="cuda")
    for kappa in (0.0, 0.5):
        loss, grad, stats = api.policy_loss_clipped(z, act, -one, one, pack(legal), zr, kl_coef=kappa, entropy_coef=0.1)
        bad = torch.arange(n, device="cuda") % 3 == 0
        assert torch.isnan(loss[bad]).all() and torch.isnan(grad[bad]).all() and torch.isnan(stats[bad, 2]).all()
        assert torch.isfinite(loss[~bad]).all() and torch.isfinite(grad[~bad]).all() and torch.isfinite(stats[~bad]).all()
    if where == "logits":
        loss, grad, stats = api.policy_loss_search(z, torch.rand((n, A), generator=g, device="cuda"), pack(legal))
        assert torch.isnan(loss[bad]).all() and torch.isnan(grad[bad]).all() and torch.isfinite(grad[~bad]).all() and torch.isfinite(loss[~bad]).all()


@pytest.mark.parametrize("A", LENGTHS)
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_largest_weights(api, dt, A):
    """Row weights up to the documented bound: actions that are not legal, or of logit -inf, still get a gradient of 0."""
    import torch
    n, T = 8, dtype_of(dt)
    rng = np.random.default_rng(A + 5)
    z, zr = [torch.from_numpy(rng.normal(0, 2, (n, A)).astype(np.float32)).to(T) for _ in range(2)]
    legal = rng.random((n, A)) < 0.6
    legal[:, 0] = True
    z[:, A // 2] = -INF
    w = np.full(n, 1e9, np.float32)
    act, one = np.zeros(n, np.int32), np.ones(n, np.float32)
    off = ~legal
    off[:, A // 2] = True
    for grad in (api.policy_loss_search(z.cuda(), cuda(rng.random((n, A)).astype(np.float32) * ~off), pack(legal), cuda(w), entropy_coef=0.2)[1],
                 api.policy_loss_clipped(z.cuda(), cuda(act), cuda(-one), cuda(one), pack(legal), zr.cuda(), cuda(w), kl_coef=0.1,
                                         entropy_coef=0.1)[1]):
        assert torch.isfinite(grad).all() and not grad.cpu()[torch.from_numpy(off)].any() and grad[:, 0].all()
