"""Policy losses and their gradients against the definitions in 64 bits: row lengths around the kernels' borders, masks that
leave one action or none, rows that are left out, values at places that are not to be looked at, strides and alignments."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


def dtype_of(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def place(x, pad, shift, fill):
    """x in rows `pad` elements further apart, `shift` elements off an aligned address; `fill` around it."""
    import torch
    n, A = x.shape
    flat = torch.full((n * (A + pad) + shift + 16,), fill, dtype=x.dtype, device="cuda")
    view = flat[shift:shift + n * (A + pad)].view(n, A + pad)[:, :A]
    view.copy_(x)
    return view, flat


def pack(legal):
    import torch
    n, A = legal.shape
    bits = np.zeros((n, (A + 31) // 32 * 32), np.uint8)
    bits[:, :A] = legal
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32).reshape(n, -1).copy()).cuda()


def make_legal(rng, n, A, mask):
    if mask == "all":
        return np.ones((n, A), bool)
    if mask == "random":
        legal = rng.random((n, A)) < rng.uniform(0.2, 1.0, (n, 1))
    else:                              # "odd": rows with one action, with none, with the last one alone
        legal = rng.random((n, A)) < 0.5
        legal[0::3] = False
        legal[1::3] = False
        legal[1::3, A - 1] = True
    return legal


def log_softmax64(z, legal):
    z = np.where(legal & (z != -np.inf), z, -np.inf)
    m = z.max(1, keepdims=True)
    m = np.where(m == -np.inf, 0.0, m)
    with np.errstate(divide="ignore"):
        lse = m + np.log(np.exp(z - m).sum(1, keepdims=True))
    return np.where(np.isfinite(z), z - np.where(np.isfinite(lse), lse, 0.0), -np.inf), lse[:, 0]


def ref_search(z, legal, t, w, beta):
    logp, lse = log_softmax64(z, legal)
    legal = np.isfinite(logp)
    p = np.exp(logp)
    lp = np.where(legal, logp, 0.0)
    t = np.where(legal, t, 0.0)
    T = t.sum(1)
    live = (T > 0) & (w != 0)
    pi = t / np.where(T > 0, T, 1.0)[:, None]
    ce, H = -(pi * lp).sum(1), -(p * lp).sum(1)
    terms = w[:, None] * (p * (1 + beta * (np.abs(lp) + H[:, None])) + pi)
    grad = w[:, None] * (p - pi + beta * p * (lp + H[:, None]))
    zero = ~live
    loss = np.where(zero, 0.0, w * (ce - beta * H))
    stats = np.stack([ce, H, T, np.where(live, lse, 0.0)], 1)
    return loss, np.where(zero[:, None], 0.0, grad), np.where(zero[:, None], 0.0, stats), terms


def ref_clipped(z, legal, action, old, adv, zr, w, lo, hi, kappa, beta):
    n, A = z.shape
    logp, _ = log_softmax64(z, legal)
    legal = np.isfinite(logp)
    rows = np.arange(n)
    inside = (action >= 0) & (action < A)
    a = np.where(inside, action, 0)
    live = inside & legal[rows, a] & (w != 0)
    p, lp = np.exp(logp), np.where(legal, logp, 0.0)
    la = lp[rows, a]
    ratio = np.exp(la - old)
    free, held = ratio * adv, np.clip(ratio, 1 - lo, 1 + hi) * adv
    c = np.where(free <= held, -free, 0.0)
    H = -(p * lp).sum(1)
    kl = np.zeros(n)
    x = np.zeros_like(z)
    if zr is not None:
        lq, _ = log_softmax64(zr, legal)
        x = np.where(legal & (p > 0), lp - lq, 0.0)
        kl = (p * x).sum(1)
    grad = -c[:, None] * p + kappa * p * (x - kl[:, None]) + beta * p * (lp + H[:, None])
    grad[rows, a] += c
    terms = p * (1 + np.abs(c)[:, None] + kappa * (np.abs(x) + np.abs(kl)[:, None] + 1) + beta * (np.abs(lp) + H[:, None] + 1))
    terms[rows, a] += np.abs(c)
    loss = w * (-np.minimum(free, held) + kappa * kl - beta * H)
    stats = np.stack([la, ratio, kl, H], 1)
    off = ~live
    return (np.where(off, 0.0, loss), np.where(off[:, None], 0.0, w[:, None] * grad), np.where(off[:, None], 0.0, stats),
            np.abs(w)[:, None] * terms, np.abs(w) * (np.abs(c) + kappa * (1 + (p * np.abs(x)).sum(1)) + beta * (1 + H)))


def relative_bound(A, reach):
    """Relative error of a probability.  exp: the difference z - M and its product with log2 e are rounded (2^-24 each of at
    most `reach`, 1.45 of them in the exponent), 2^-22 for the hardware's power of two; the sum adds A / 32 terms per lane
    and 10 joins, each join scaling by such a power: 2^-24 and 2^-22 a piece; twice, for numerator and sum, and once more
    for the reciprocal and the products behind it."""
    e = 2 * 1.45 * reach * 2.0 ** -24 + 2.0 ** -22
    return 2 * e + (A / 32 + 10) * 2.0 ** -24 + 10 * 2.0 ** -22 + 8 * 2.0 ** -24


def half_step(dt):
    import torch
    return torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


SIZES = [(1, 1), (1, 2), (5, 31), (4, 32), (9, 33), (3, 127), (300, 225), (37, 362), (3, 511), (3, 513), (4, 1023), (3, 1024),
         (5, 1025), (3, 2049), (70, 4672), (2, 8191), (2, 8193), (1, 16384), (2, 32769), (1, 65536), (1, 65537), (2, 150001), (3, 300007)]


@pytest.mark.parametrize("n,A", SIZES)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("mask,target,pad,shift", [("all", "visits", 0, 0), ("random", "probs", 3, 1), ("odd", "visits", 8, 0), ("random", "probs", 0, 0)])
def test_search_loss(api, n, A, dt, mask, target, pad, shift):
    import torch
    rng = np.random.default_rng(n * 1000003 + A * 17 + len(mask) + pad)
    T = dtype_of(dt)
    z = torch.from_numpy(rng.normal(0, 3, (n, A)).astype(np.float32)).to(T)
    legal = make_legal(rng, n, A, mask)
    w = rng.uniform(0.5, 2.0, n).astype(np.float32)
    if n > 2:
        w[n // 2] = 0
    if target == "visits":
        t = rng.poisson(2.0, (n, A)).astype(np.int32)
        if n > 3:
            t[3] = 0
        tt = torch.from_numpy(t)
    else:
        t = rng.gamma(0.3, 1.0, (n, A)).astype(np.float32)
        tt = torch.from_numpy(t)
    z64 = z.double().numpy()
    if mask != "all":                  # what is not legal is not looked at
        bad = torch.from_numpy(~legal)
        z[bad] = float("nan")
        z[:, ::2][bad[:, ::2]] = float("inf")
        if target == "probs":
            tt[bad] = float("nan")
    zd, zflat = place(z.cuda(), pad, shift, 7.0)
    td, _ = place(tt.cuda(), pad, shift, 5)
    gd, gflat = place(torch.full((n, A), 9.0, dtype=T).cuda(), pad, shift, 11.0)
    loss = torch.full((n,), 7.0, device="cuda")
    stats = torch.full((n, 4), 7.0, device="cuda")
    bits = None if mask == "all" else pack(legal)
    before = zflat.clone()
    api.policy_loss_search(zd, td, bits, torch.from_numpy(w).cuda(), entropy_coef=0.05, out=(loss, gd, stats))
    torch.cuda.synchronize()
    rl, rg, rs, terms = ref_search(z64, legal, t.astype(np.float64), w.astype(np.float64), 0.05)
    reach = 2 * np.abs(z64).max() + 1
    D = relative_bound(A, reach)
    half, least = half_step(T)
    g = gd.double().cpu().numpy()
    tol = 4 * D * terms + half * np.abs(rg) + least
    assert (np.abs(g - rg) <= tol).all(), float((np.abs(g - rg) / tol).max())
    assert (g[~legal] == 0).all()
    stol = 4 * D * (1 + reach + np.abs(rs))
    assert (np.abs(stats.double().cpu().numpy() - rs) <= stol).all()
    ltol = 4 * D * (np.abs(rl) + w * (1 + 0.05) * (1 + reach))
    assert (np.abs(loss.double().cpu().numpy() - rl) <= ltol).all()
    # inputs and everything around the gradient stay as they were
    assert torch.equal(zflat.view(torch.int16 if T != torch.float32 else torch.int32), before.view(torch.int16 if T != torch.float32 else torch.int32))
    around = gflat.clone()
    around[shift:shift + n * (A + pad)].view(n, A + pad)[:, :A] = 11.0
    assert (around == 11.0).all()


@pytest.mark.parametrize("n,A", SIZES)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("mask,ref,pad,shift", [("all", True, 0, 0), ("random", True, 3, 1), ("odd", True, 8, 0), ("random", False, 0, 0)])
def test_clipped_loss(api, n, A, dt, mask, ref, pad, shift):
    import torch
    rng = np.random.default_rng(n * 1000003 + A * 19 + len(mask) + pad)
    T = dtype_of(dt)
    z = torch.from_numpy(rng.normal(0, 3, (n, A)).astype(np.float32)).to(T)
    zr = (z.float() + torch.from_numpy(rng.normal(0, 0.5, (n, A)).astype(np.float32))).to(T)
    legal = make_legal(rng, n, A, mask)
    w = rng.uniform(0.5, 2.0, n).astype(np.float32)
    if n > 2:
        w[n // 2] = 0
    z64, zr64 = z.double().numpy(), zr.double().numpy()
    action = np.array([rng.choice(np.nonzero(row)[0]) if row.any() else 0 for row in legal], np.int32)
    if n > 4:
        action[2], action[4] = -1, A             # left out
    logp, _ = log_softmax64(z64, legal)
    la = logp[np.arange(n), np.clip(action, 0, A - 1)]
    d = rng.choice([-0.5, -0.1, 0.0, 0.1, 0.4], n) + rng.uniform(-0.02, 0.02, n)      # away from the clip's borders
    old = (np.where(np.isfinite(la), la, 0.0) - d).astype(np.float32)
    adv = rng.normal(0, 1, n).astype(np.float32)
    if n > 5:
        adv[5] = 0
    if mask != "all":
        bad = torch.from_numpy(~legal)
        z[bad] = float("nan")
        zr[bad] = float("inf")
    zd, _ = place(z.cuda(), pad, shift, 7.0)
    rd, _ = place(zr.cuda(), pad, shift, 5.0)
    gd, gflat = place(torch.full((n, A), 9.0, dtype=T).cuda(), pad, shift, 11.0)
    loss = torch.full((n,), 7.0, device="cuda")
    stats = torch.full((n, 4), 7.0, device="cuda")
    kappa = 0.2 if ref else 0.0
    cuda = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    api.policy_loss_clipped(zd, cuda(action), cuda(old), cuda(adv), None if mask == "all" else pack(legal), rd if ref else None, cuda(w),
                            clip_low=0.2, clip_high=0.25, kl_coef=kappa, entropy_coef=0.05, out=(loss, gd, stats))
    torch.cuda.synchronize()
    rl, rg, rs, terms, lterm = ref_clipped(z64, legal, action, old.astype(np.float64), adv.astype(np.float64), zr64 if ref else None,
                                           w.astype(np.float64), 0.2, 0.25, kappa, 0.05)
    reach = 2 * max(np.abs(z64).max(), np.abs(zr64).max()) + 1
    D = relative_bound(A, reach)
    half, least = half_step(T)
    g = gd.double().cpu().numpy()
    # the ratio's error: that of a log-probability, reach * 2^-23 + D, and of its exp
    tol = (4 * D + reach * 2.0 ** -22) * terms + half * np.abs(rg) + least
    assert (np.abs(g - rg) <= tol).all(), float((np.abs(g - rg) / tol).max())
    assert (g[~legal] == 0).all()
    E = 4 * D * (1 + reach)
    stol = E * (1 + np.abs(rs))
    assert (np.abs(stats.double().cpu().numpy() - rs) <= stol).all(), float((np.abs(stats.double().cpu().numpy() - rs) / stol).max())
    assert (np.abs(loss.double().cpu().numpy() - rl) <= E * (np.abs(rl) + lterm + np.abs(w))).all()
    around = gflat.clone()
    around[shift:shift + n * (A + pad)].view(n, A + pad)[:, :A] = 11.0
    assert (around == 11.0).all()


@pytest.mark.parametrize("A", [7, 225, 1030, 9000])
@pytest.mark.parametrize("kind", ["search", "clipped"])
def test_gradient_against_differences(api, A, kind):
    """The gradient is the loss's: central differences of the kernel's own loss, in random directions."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(A)
    n = 6
    z = torch.randn((n, A), generator=g, device="cuda")
    zr = z + 0.5 * torch.randn((n, A), generator=g, device="cuda")
    t = torch.rand((n, A), generator=g, device="cuda")
    act = torch.randint(0, A, (n,), generator=g, device="cuda").int()
    old = torch.log_softmax(z, 1).gather(1, act.long()[:, None])[:, 0] - 0.05
    adv = torch.randn(n, generator=g, device="cuda")
    v = torch.randn((n, A), generator=g, device="cuda")

    def loss(x):
        if kind == "search":
            return api.policy_loss_search(x, t, entropy_coef=0.1)
        return api.policy_loss_clipped(x, act, old, adv, ref_logits=zr, kl_coef=0.3, entropy_coef=0.1)
    h = 2.0 ** -7
    up, down = loss(z + h * v)[0].double(), loss(z - h * v)[0].double()
    along = (loss(z)[1].double() * v.double()).sum(1)
    # h^2 / 6 of the third derivative along v (below 2 + |adv| for weights of order 1, |v| concentrated on p), and two losses'
    # rounding (of order 10 each, 2^-20 relative) over 2 h
    tol = h * h * (4 + 4 * adv.abs().double()) + 2 * 10 * 2.0 ** -20 / (2 * h)
    assert ((up - down) / (2 * h) - along).abs().le(tol).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("A", [33, 225, 4672, 40000, 300007])
def test_lowest_values_and_infinities(api, dt, A):
    import torch
    T = dtype_of(dt)
    low = torch.finfo(T).min
    z = torch.zeros((5, A), dtype=T)
    z[0] = low                           # all at the lowest value: uniform
    z[1] = low
    z[1, A // 2] = 1.0                   # one above it
    z[2] = -float("inf")                 # no action
    z[3, 1:] = -float("inf")             # one action
    z[4, 3] = float("nan")               # a NaN counts
    t = torch.ones((5, A))
    t[3, 1:] = 0
    loss, grad, stats = api.policy_loss_search(z.cuda(), t.cuda())
    torch.cuda.synchronize()
    grad, stats = grad.double().cpu(), stats.double().cpu()
    D = relative_bound(A, 1)
    assert abs(float(stats[0, 1]) - math.log(A)) <= 4 * D * (1 + math.log(A))
    assert grad[0].abs().max() <= 4 * D * 2 / A + torch.finfo(T).eps / 2 * 4 * D
    assert abs(float(grad[1, A // 2]) - (1 - 1 / A)) <= 4 * D + torch.finfo(T).eps / 2
    assert float(loss[2]) == 0 and not grad[2].any() and not stats[2].any()
    assert float(loss[3]) == 0 and not grad[3].any() and float(stats[3, 2]) == 1
    assert math.isnan(float(loss[4])) and torch.isnan(grad[4]).all()


def test_all_rows_left_out_and_no_rows(api):
    import torch
    z = torch.full((4, 225), float("nan"), device="cuda")
    loss, grad, stats = api.policy_loss_search(z, torch.ones((4, 225), device="cuda"), row_weight=torch.zeros(4, device="cuda"))
    assert not loss.any() and not grad.any() and not stats.any()
    loss, grad, stats = api.policy_loss_search(z[:0], torch.ones((0, 225), device="cuda"))
    assert grad.shape == (0, 225)
    e = torch.empty(0, device="cuda")
    api.policy_loss_clipped(z[:0], e.int(), e, e)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("A", [225, 1000, 4672, 32768, 70000, 300007])
def test_gradient_in_place(api, dt, A):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(A)
    z = torch.randn((9, A), generator=g, device="cuda").to(dtype_of(dt))
    zr = torch.randn((9, A), generator=g, device="cuda").to(dtype_of(dt))
    act = torch.randint(0, A, (9,), generator=g, device="cuda").int()
    old, adv = torch.zeros(9, device="cuda") - 5, torch.randn(9, generator=g, device="cuda")
    want = api.policy_loss_clipped(z, act, old, adv, ref_logits=zr, kl_coef=0.1, entropy_coef=0.1)
    x = z.clone()
    got = api.policy_loss_clipped(x, act, old, adv, ref_logits=zr, kl_coef=0.1, entropy_coef=0.1,
                                  out=(torch.empty_like(want[0]), x, torch.empty_like(want[2])))
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_optional_outputs_streams_and_graph(api):
    """loss and stats may be left out; a call on a stream of its own, captured and replayed on new inputs."""
    import torch
    z = torch.randn((64, 225), device="cuda")
    t = torch.rand((64, 225), device="cuda")
    want = api.policy_loss_search(z, t)[1].clone()
    grad = torch.empty_like(z)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        api.policy_loss_search(z, t, out=(None, grad, None))
    s.synchronize()
    assert torch.equal(grad, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.policy_loss_search(z, t, out=(None, grad, None))
    z.copy_(torch.randn((64, 225), device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, api.policy_loss_search(z, t)[1])


@pytest.mark.parametrize("A", [225, 1030, 40000])
def test_many_rows_of_each_kind(api, A):
    """More rows than teams: rows of weight 0, without a legal action, with a single one, at the lowest value alone, in turn,
    against the definition in 64 bits for a few of each."""
    import torch
    n = 40000 if A == 225 else 3000 if A == 1030 else 700
    g = torch.Generator(device="cuda")
    g.manual_seed(A)
    z = torch.randn((n, A), generator=g, device="cuda").mul_(3).bfloat16()
    t = torch.rand((n, A), generator=g, device="cuda")
    legal = torch.rand((n, A), generator=g, device="cuda") < 0.6
    w = torch.ones(n, device="cuda")
    kind = torch.arange(n, device="cuda") % 7
    w[kind == 1] = 0
    legal[kind == 2] = False
    legal[kind == 3] = False
    legal[kind == 3, A // 3] = True
    z[kind == 4] = torch.finfo(torch.bfloat16).min
    z[kind == 5] = -float("inf")
    loss, grad, stats = api.policy_loss_search(z, t, pack(legal.cpu().numpy()), w, entropy_coef=0.1)
    torch.cuda.synchronize()
    for k in (1, 2, 5):
        assert not loss[kind == k].any() and not grad[kind == k].any() and not stats[kind == k].any()
    assert not grad[~legal].any()
    rows = torch.cat([(kind == k).nonzero()[[0, 1, -1], 0] for k in (0, 3, 4, 6)])
    z64 = np.where(kind.cpu().numpy()[rows.cpu().numpy(), None] == 4, 0.0, z[rows].double().cpu().numpy())      # all alike: the same policy
    rl, rg, rs, terms = ref_search(z64, legal[rows].cpu().numpy(), t[rows].double().cpu().numpy(), np.ones(len(rows)), 0.1)
    reach = 2 * np.abs(z64).max() + 1
    D = relative_bound(A, reach)
    half, least = half_step(torch.bfloat16)
    assert (np.abs(grad[rows].double().cpu().numpy() - rg) <= 4 * D * terms + half * np.abs(rg) + least).all()
    got = stats[rows].double().cpu().numpy()
    assert (np.abs(got - rs)[:, :3] <= 4 * D * (1 + reach + np.abs(rs[:, :3]))).all()


def test_more_rows_than_a_grid_dimension(api):
    """Offsets beyond 2^31 elements: the last rows of a matrix of 2.2e9 (4.4 GB twice)."""
    import torch
    n, A = 70000, 31500
    z = torch.zeros((n, A), dtype=torch.bfloat16, device="cuda")
    z[-1, :] = torch.randn(A, device="cuda")
    w = torch.zeros(n, device="cuda")
    w[0] = w[-1] = 1.0
    act = torch.full((n,), 5, dtype=torch.int32, device="cuda")
    old = torch.full((n,), -9.0, device="cuda")
    loss, _, stats = api.policy_loss_clipped(z, act, old, torch.ones(n, device="cuda"), row_weight=w, out=(torch.empty(n, device="cuda"), z, torch.empty((n, 4), device="cuda")))
    torch.cuda.synchronize()
    assert abs(float(stats[0, 3]) - math.log(A)) < 1e-3 and 0 < float(stats[-1, 3]) < math.log(A) - 0.1
    assert not z[1:-1].any() and z[-1].any()


@pytest.mark.parametrize("A", [225, 4672, 40000, 300007])
def test_two_calls_at_once(api, A):
    """Calls on two streams at the same time give what each gives alone."""
    import torch
    n = max(8, 4000000 // A)
    torch.manual_seed(A)
    zs = [torch.randn((n + k, A), device="cuda").bfloat16() for k in (0, 5)]
    acts = [torch.randint(0, A, (z.shape[0],), device="cuda").int() for z in zs]
    ones = [torch.ones(z.shape[0], device="cuda") for z in zs]

    def call(k, out=None):
        return api.policy_loss_clipped(zs[k], acts[k], -ones[k], ones[k], ref_logits=refs[k], kl_coef=0.1, out=out)
    refs = [z.flip(1) for z in zs]
    want = [call(0), call(1)]
    outs = [[tuple(torch.zeros_like(x) for x in w) for _ in range(8)] for w in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in zs]
    for i in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                call(k, outs[k][i])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for w, rounds in zip(want, outs) for got in rounds for x, y in zip(got, w))
