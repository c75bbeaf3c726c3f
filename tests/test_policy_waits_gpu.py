"""What the policy losses and a learner leave when a kernel's bounded wait runs out: made to by a hook that lets every wait run
out at once; nothing hangs and the context stays usable."""
import pytest

from test_learn_gpu import batch, make
from test_policy_loss_gpu import TYPES, dtype_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


@pytest.fixture
def no_waits(api):
    import torch
    torch.cuda.synchronize()
    assert api.device_error_code() == 0
    api.lib().ob200_debug_policy_waits(1)
    yield
    api.lib().ob200_debug_policy_waits(0)
    torch.cuda.synchronize()
    api.device_error_code()


@pytest.mark.parametrize("n,A", [(3, 225), (40000, 225), (9000, 1000), (700, 4672), (40, 40000), (3, 40000), (200, 100000)])
@pytest.mark.parametrize("dt", TYPES)
def test_rows_without_their_copies_are_nan(api, no_waits, n, A, dt):
    import torch
    T = dtype_of(dt)
    z = torch.randn((n, A), device="cuda").to(T)
    w = torch.ones(n, device="cuda")
    w[1] = 0
    act, adv = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.ones(n, device="cuda")
    for call in (lambda: api.policy_loss_search(z, torch.rand((n, A), device="cuda"), None, w),
                 lambda: api.policy_loss_clipped(z, act, -adv, adv, None, z, w, kl_coef=0.1)):
        loss, grad, stats = call()
        torch.cuda.synchronize()
        assert api.device_error_code() == 4
        alive = w != 0
        for x in (loss, grad, stats):
            assert torch.isnan(x[alive]).all() and not x[1].any()
        norm = api.GradNorm([grad]).run(1.0)
        assert torch.isnan(norm[1])


def test_calls_afterwards_are_as_ever(api):
    import torch
    z, t = torch.randn((300, 4672), device="cuda"), torch.rand((300, 4672), device="cuda")
    want = api.policy_loss_search(z, t)
    torch.cuda.synchronize()
    api.lib().ob200_debug_policy_waits(1)
    api.policy_loss_search(z, t)
    api.lib().ob200_debug_policy_waits(0)
    got = api.policy_loss_search(z, t)
    torch.cuda.synchronize()
    assert api.device_error_code() == 4 and all(torch.equal(a, b) for a, b in zip(want, got))


def test_learner_reports_and_leaves_the_step_out(api, no_waits):
    import torch
    net, w, learner = make(api)
    b, _ = batch(40)
    before = {k: p.detach().clone() for k, p in learner.params.items()}
    record = {"moves": [0, 1, 2], "winner": 1, "policies": [[1.0] * 225] * 3}
    for ask in (lambda: learner.weights(), lambda: learner.fit([record], steps=0), lambda: learner.fit([record], steps=2, batch=8)):
        loss, _, _, norm = learner.step_search(b["history"], b["n_hist"], b["to_move"], b["visits"], b["outcome"], b["legal_bits"])
        with pytest.raises(api.Error) as e:
            ask()
        assert e.value.code == api.ERR_TIMEOUT
        with pytest.raises(api.Error):           # it is there for the others on the device too
            learner.weights()
        assert api.device_error_code(clear=False) == 4 == api.device_error_code() and api.device_error_code() == 0
        assert torch.isnan(loss).all() and torch.isnan(norm[1])
        assert all(torch.equal(p, before[k]) for k, p in learner.params.items())
    api.lib().ob200_debug_policy_waits(0)
    learner.step_search(b["history"], b["n_hist"], b["to_move"], b["visits"], b["outcome"], b["legal_bits"])
    assert learner.weights() and not torch.equal(learner.params["policy_fc.weight"], before["policy_fc.weight"])
