"""Policy losses, the kernels' own borders: matrices that do not lie alike within 16 bytes, and rows of many warps whose action
stands in any one of them."""
import numpy as np
import pytest

from test_policy_loss_gpu import (SIZES, TYPES, dtype_of, half_step, log_softmax64, make_legal, pack, place, ref_clipped, ref_search,
                                  relative_bound)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


def within(got, want, tol):
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), float((err / tol).max())


# (pad, shift) of the logits, of the other matrix, of the gradient: the first columns of a wider output with the rest
# contiguous; one pitch and three starts; a gradient alone that is off
UNLIKE = [((5, 0), (0, 0), (0, 0)), ((8, 1), (8, 2), (8, 0)), ((0, 0), (0, 0), (3, 1))]


@pytest.mark.parametrize("places", UNLIKE, ids=["columns", "starts", "gradient"])
@pytest.mark.parametrize("n,A", [s for s in SIZES if s != (1, 1)])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kind", ["visits", "probs", "clipped", "reference"])
def test_matrices_that_do_not_lie_alike(api, n, A, dt, kind, places):
    """Sizes, masks and bounds of the tests of matrices that do."""
    import torch
    rng = np.random.default_rng(n * 1000003 + A * 23 + len(kind))
    T = dtype_of(dt)
    (zp, zs), (xp, xs), (gp, gs) = places
    if n == 1 and zs == xs == gs:
        zs = 1                                   # a single row's pitch does not count
    z = torch.from_numpy(rng.normal(0, 3, (n, A)).astype(np.float32)).to(T)
    mask = ["all", "random", "odd"][(n + A + len(kind)) % 3]
    legal = make_legal(rng, n, A, mask)
    w = rng.uniform(0.5, 2.0, n).astype(np.float32)
    if n > 2:
        w[n // 2] = 0
    z64 = z.double().numpy()
    bad = torch.from_numpy(~legal)
    z[bad] = float("nan")
    bits = None if mask == "all" else pack(legal)
    cuda = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    zd, _ = place(z.cuda(), zp, zs, 7.0)
    gd, gflat = place(torch.full((n, A), 9.0, dtype=T).cuda(), gp, gs, 11.0)
    out = (torch.full((n,), 7.0, device="cuda"), gd, torch.full((n, 4), 7.0, device="cuda"))
    half, least = half_step(T)
    if kind in ("visits", "probs"):
        t = rng.poisson(2.0, (n, A)).astype(np.int32) if kind == "visits" else rng.gamma(0.3, 1.0, (n, A)).astype(np.float32)
        td, _ = place(cuda(t), xp, xs, 5)
        api.policy_loss_search(zd, td, bits, cuda(w), entropy_coef=0.05, out=out)
        rl, rg, rs, terms = ref_search(z64, legal, t.astype(np.float64), w.astype(np.float64), 0.05)
        reach = 2 * np.abs(z64).max() + 1
        D = relative_bound(A, reach)
        within(gd, rg, 4 * D * terms + half * np.abs(rg) + least)
        within(out[2], rs, 4 * D * (1 + reach + np.abs(rs)))
        within(out[0], rl, 4 * D * (np.abs(rl) + w * 1.05 * (1 + reach)))
    else:
        zr = (z.float().nan_to_num(0.0) + torch.from_numpy(rng.normal(0, 0.5, (n, A)).astype(np.float32))).to(T)
        zr64 = zr.double().numpy()
        zr[bad] = float("inf")
        ref = kind == "reference"
        kappa = 0.2 if ref else 0.0
        action = np.array([rng.choice(np.nonzero(row)[0]) if row.any() else 0 for row in legal], np.int32)
        la = log_softmax64(z64, legal)[0][np.arange(n), action]
        d = rng.choice([-0.5, -0.1, 0.0, 0.1, 0.4], n) + rng.uniform(-0.02, 0.02, n)
        old = (np.where(np.isfinite(la), la, 0.0) - d).astype(np.float32)
        adv = rng.normal(0, 1, n).astype(np.float32)
        rd, _ = place(zr.cuda(), xp, xs, 5.0)
        api.policy_loss_clipped(zd, cuda(action), cuda(old), cuda(adv), bits, rd if ref else None, cuda(w), clip_low=0.2, clip_high=0.25,
                                kl_coef=kappa, entropy_coef=0.05, out=out)
        rl, rg, rs, terms, lterm = ref_clipped(z64, legal, action, old.astype(np.float64), adv.astype(np.float64), zr64 if ref else None,
                                               w.astype(np.float64), 0.2, 0.25, kappa, 0.05)
        reach = 2 * max(np.abs(z64).max(), np.abs(zr64).max()) + 1
        D = relative_bound(A, reach)
        E = 4 * D * (1 + reach)
        within(gd, rg, (4 * D + reach * 2.0 ** -22) * terms + half * np.abs(rg) + least)
        within(out[2], rs, E * (1 + np.abs(rs)))
        within(out[0], rl, E * (np.abs(rl) + lterm + np.abs(w)))
    assert not gd.cpu()[bad].any()
    around = gflat.clone()
    around[gs:gs + n * (A + gp)].view(n, A + gp)[:, :A] = 11.0
    assert (around == 11.0).all()


@pytest.mark.parametrize("at", ["first", "middle", "last"])
@pytest.mark.parametrize("A", [225, 1025, 4667, 4672, 9001, 30000])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shift", [(0, 0), (1, 1), (0, 1)], ids=["aligned", "alike", "unlike"])
def test_rows_of_one_content_get_one_result(api, A, dt, at, shift):
    """Every warp of a row takes the action's logit, not what stands in its place once another warp has written its
    gradient: thousands of rows with the same content have the same loss, statistics and gradient, bit by bit."""
    import torch
    T = dtype_of(dt)
    n = min(4096, (1 << 25) // A)
    pitch = (A + 7) // 8 * 8                     # rows start alike
    g = torch.Generator(device="cuda")
    g.manual_seed(A)
    row, ref = torch.randn((2, A), generator=g, device="cuda").to(T)
    a = {"first": 0, "middle": A // 2 + 1, "last": A - 1}[at]

    def matrix(s, content):
        x = torch.zeros(n * pitch + 16, dtype=T, device="cuda")[s:s + n * pitch].view(n, pitch)[:, :A]
        return x.copy_(content.expand(n, A))
    act = torch.full((n,), a, dtype=torch.int32, device="cuda")
    old = torch.log_softmax(row.float(), 0)[a].expand(n).contiguous() - 0.1
    for zr in (None, matrix(shift[0], ref)):
        out = (torch.zeros(n, device="cuda"), matrix(shift[1], torch.zeros_like(row)), torch.zeros((n, 4), device="cuda"))
        api.policy_loss_clipped(matrix(shift[0], row), act, old, torch.ones(n, device="cuda"), ref_logits=zr, kl_coef=0.1 if zr is not None else 0.0,
                                entropy_coef=0.01, out=out)
        for x in out:
            assert torch.equal(x, x[:1].expand_as(x))
        # the ratio is exp(0.1): not clipped, so the action is to become likelier
        assert abs(float(out[2][0, 1]) - 1.10517) < 1e-3 and float(out[1][0, a]) < 0
