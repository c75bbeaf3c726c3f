"""The learner's steps on the device: gradients of the heads against the same objective in plain fp64 PyTorch, one step's
weights against AdamW in fp64, self-play records through to a new handle."""
import numpy as np
import pytest

from omoknuni_small_b200 import synth

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


def make(api, B=64, S=15, dtype=0, **kw):
    from omoknuni_small_b200 import learn
    shapes = synth.net_tensor_shapes(S, 17, 64, 2, S * S, 4, 2, value_hidden=32)
    w = synth.make_weights(shapes, seed=3, init="torch_default", bn="random")
    net = api.Net(17, S, 2, 64, S * S, 4, 2, 32, B, tower_dtype=dtype).load(w)
    return net, w, learn.HeadLearner(net, w, **kw)


def batch(n, S=15, seed=1):
    import torch
    games, hist, nh, tm = synth.make_gomoku_games(n, S, seed=seed)
    rng = np.random.default_rng(seed)
    legal = np.ones((n, (S * S + 31) // 32 * 32), np.uint8)
    legal[:, S * S:] = 0
    for i, g in enumerate(games):
        legal[i, np.asarray(g, np.int64)] = 0
    bits = np.packbits(legal, axis=1, bitorder="little").view(np.int32).reshape(n, -1)
    visits = rng.poisson(3.0, (n, S * S)).astype(np.int32)
    out = dict(history=hist, n_hist=nh, to_move=tm, legal_bits=bits.copy(), visits=visits, outcome=rng.choice([-1.0, 0.0, 1.0], n).astype(np.float32))
    return {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in out.items()}, legal[:, :S * S].astype(bool)


def heads64(torch, x, p, fixed):
    def branch(name):
        y = torch.einsum("nfyx,cf->ncyx", x, p[name + "_conv.weight"][:, :, 0, 0])
        s = p[name + "_bn.weight"] / torch.sqrt(fixed[name + "_bn.running_var"].double() + 1e-5)
        y = (y - fixed[name + "_bn.running_mean"].double()[:, None, None]) * s[:, None, None] + p[name + "_bn.bias"][:, None, None]
        return y.relu().flatten(1)
    logits = branch("policy") @ p["policy_fc.weight"].t() + p["policy_fc.bias"]
    v = (branch("value") @ p["value_fc1.weight"].t() + p["value_fc1.bias"]).relu()
    return logits, torch.tanh(v @ p["value_fc2.weight"].t() + p["value_fc2.bias"]).flatten()


@pytest.mark.parametrize("dtype", [0, 1], ids=["bf16", "f16"])
@pytest.mark.parametrize("objective", ["search", "clipped"])
def test_gradients_and_update(api, dtype, objective):
    import torch
    n = 48
    net, w, learner = make(api, dtype=dtype, entropy_coef=0.01, max_norm=0.05, weight_decay=0.1)
    b, legal = batch(n)
    x = learner.features(b["history"], b["n_hist"], b["to_move"]).double()
    p = {k: v.detach().double().requires_grad_(True) for k, v in learner.params.items()}
    logits, value = heads64(torch, x, p, learner.fixed)
    lg = torch.from_numpy(legal).cuda()
    lp = torch.log_softmax(logits.masked_fill(~lg, -float("inf")), 1)
    safe = torch.where(lg, lp, torch.zeros_like(lp))
    prob = torch.where(lg, lp.exp(), torch.zeros_like(lp))
    H = -(prob * safe).sum(1)
    if objective == "search":
        t = torch.where(lg, b["visits"].double(), torch.zeros_like(lp))
        row = -(t * safe).sum(1) / t.sum(1)
    else:
        torch.manual_seed(0)
        act = torch.where(lg, torch.rand_like(lp), torch.zeros_like(lp) - 1).argmax(1)
        adv = torch.randn(n, device="cuda")
        old = (safe.gather(1, act[:, None])[:, 0].detach() - torch.tensor([-0.5, -0.05, 0.05, 0.5], device="cuda").repeat(n // 4)).float()
        r = (safe.gather(1, act[:, None])[:, 0] - old.double()).exp()
        row = -torch.minimum(r * adv.double(), r.clamp(0.8, 1.2) * adv.double())      # the KL is 0 at the start, and so is its gradient
    total = ((row - 0.01 * H) / n).sum() + ((value - b["outcome"].double()) ** 2 / n).sum()
    want = torch.autograd.grad(total, list(p.values()))
    common = (b["history"], b["n_hist"], b["to_move"])
    if objective == "search":
        loss, vloss, stats, norm = learner.step_search(*common, b["visits"], b["outcome"], b["legal_bits"], lr=0.01)
    else:
        loss, vloss, stats, norm = learner.step_clipped(*common, act.int(), old, adv, b["outcome"], b["legal_bits"], kl_coef=0.3, lr=0.01)
    torch.cuda.synchronize()
    assert abs(float(loss.double().sum() + vloss.double().sum()) - float(total.detach())) <= 1e-5 * (1 + abs(float(total.detach())))
    size = torch.sqrt(sum((g * g).sum() for g in want))
    # fp32 heads: sums of at most 900 products forward and 10,800 backward, each 2^-24 of its terms, which are of the size of
    # the result or, where they cancel, of the whole gradient: sqrt(10,800) 2^-24 = 6e-6, taken 30 times over
    for (k, q), g in zip(learner.params.items(), want):
        assert float((q.grad.double() - g).norm()) <= 2e-4 * float(g.norm() + 0.01 * size), k
    assert abs(float(norm[0]) - float(size)) <= 2e-4 * float(size)
    scale = min(1.0, 0.05 / float(norm[0]))
    for k, q in learner.params.items():
        g = q.grad.double() * scale
        old_p = torch.from_numpy(w[k]).cuda().double()
        step = 0.01 * g / (g.abs() + 1e-8)                    # the first step: m and v's factors cancel
        decay = 0.1 if q.dim() > 1 else 0.0
        new = old_p * (1 - 0.01 * decay) - step
        assert ((q.detach().double() - new).abs() <= 2.0 ** -20 * (0.01 + old_p.abs())).all(), k


@pytest.mark.parametrize("bits", [32, 8])
def test_records_to_a_new_handle(api, bits):
    """Self-play -> records -> steps -> weights -> a handle that answers as the learner's heads do."""
    import torch
    from omoknuni_small_b200 import selfplay
    net, w, learner = make(api, B=64, state_bits=bits)
    search = api.Search(net, n_trees=8, sims_per_move=32, leaf_batch=64, max_depth=16, seed=5)
    records = selfplay.SelfPlay(search, max_moves=8, seed=2).generate_games(8)
    losses = learner.fit(records, steps=3, batch=40, lr=1e-3, seed=4)
    assert losses.shape == (3, 2) and np.isfinite(losses).all()
    new = learner.weights()
    assert set(new) == set(w) and not np.array_equal(new["policy_fc.weight"], w["policy_fc.weight"])
    assert all(np.array_equal(new[k], w[k]) for k in w if k.startswith(("res_blocks", "input")))
    fresh = api.Net(17, 15, 2, 64, 225, 4, 2, 32, 64).load(new)
    b, _ = batch(32, seed=9)
    x = learner.features(b["history"], b["n_hist"], b["to_move"])
    logits, value = [t.detach().cpu().numpy() for t in learner.heads(x)]
    got, v = fresh.infer_gomoku(b["history"].cpu().numpy(), b["n_hist"].cpu().numpy(), b["to_move"].cpu().numpy(), api.OUT_LOGITS)
    # the same tower and the same fp32 heads, in another order of additions: 900 terms a logit
    assert np.abs(got - logits).max() <= 1e-4 * (1 + np.abs(logits).max()) and np.abs(v - value).max() <= 1e-4


def test_rows_that_fill_up_a_batch(api):
    """Rows of weight 0 change nothing whatever stands in their targets and outcomes; what a step returned stays as it was."""
    import torch
    _, _, a = make(api)
    _, _, b = make(api)
    clean, _ = batch(40)
    fill = {k: v.clone() for k, v in clean.items()}
    fill["outcome"][24:] = float("nan")
    fill["visits"][24:] = -1
    fill["legal_bits"][24:] = 0
    w = torch.full((40,), 1.0 / 24, device="cuda")
    w[24:] = 0
    args = ("history", "n_hist", "to_move", "visits", "outcome", "legal_bits")
    first = a.step_search(*[clean[k] for k in args], row_weight=w, lr=1e-3)
    kept = [t.clone() for t in first]
    got = b.step_search(*[fill[k] for k in args], row_weight=w, lr=1e-3)
    assert all(torch.isfinite(x).all() and torch.equal(x, y) for x, y in zip(got, first))
    assert not got[0][24:].any() and not got[1][24:].any() and first[0][:24].all()
    assert all(torch.equal(p, b.params[k]) for k, p in a.params.items())
    a.step_search(*[clean[k] for k in args], row_weight=w, lr=1e-3)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, kept))
    assert a.fit([{"moves": [0], "winner": 0, "policies": [[1.0] * 225]}], steps=0).shape == (0, 2)


def test_refusals(api):
    import torch
    net, w, learner = make(api, B=16)
    b, _ = batch(17)
    with pytest.raises(api.Error):
        learner.features(b["history"], b["n_hist"], b["to_move"])
    with pytest.raises(api.Error):
        learner.fit([], 1)
    from omoknuni_small_b200 import learn
    with pytest.raises(api.Error):
        learn.HeadLearner(net, {k: v for k, v in w.items() if not k.startswith("policy_fc")})
