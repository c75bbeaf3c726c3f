"""Policy losses at the ends of what the header allows: reference policies without any probability."""
import numpy as np
import pytest

from test_policy_loss_gpu import TYPES, dtype_of, half_step, pack, ref_clipped, relative_bound

pytestmark = pytest.mark.gpu

LENGTHS = [7, 225, 1000, 4672, 40000, 300007]        # lanes, warps, CTAs, clusters, clusters over device memory
INF = float("inf")


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


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
