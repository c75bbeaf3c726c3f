"""The learner on networks of each tower kernel: its heads answer as the handle does, before a step and, in a new handle,
after it."""
import numpy as np
import pytest

from omoknuni_small_b200 import synth
from test_learn_gpu import batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


# filters, board, planes, policy and value head channels: one launch of resident boards, a launch per layer, streamed
# weights, boards of eight
@pytest.mark.parametrize("F,S,planes,pc,vc", [(64, 9, 19, 2, 1), (64, 15, 17, 32, 32), (64, 19, 17, 2, 2), (128, 13, 17, 4, 1), (256, 15, 19, 2, 2),
                                              (256, 8, 17, 3, 2), (128, 8, 17, 2, 1)])
@pytest.mark.parametrize("dtype", [0, 1], ids=["bf16", "f16"])
def test_step_on_each_tower(api, F, S, planes, pc, vc, dtype):
    import torch
    from omoknuni_small_b200 import learn
    n = 37
    shapes = synth.net_tensor_shapes(S, planes, F, 2, S * S, pc, vc, value_hidden=32)
    w = synth.make_weights(shapes, seed=3, init="torch_default", bn="random")

    def handle(weights):
        return api.Net(planes, S, 2, F, S * S, pc, vc, 32, 64, tower_dtype=dtype).load(weights)
    net = handle(w)
    learner = learn.HeadLearner(net, w, max_norm=0.5)
    b, legal = batch(n, S)
    args = (b["history"], b["n_hist"], b["to_move"])
    host = [t.cpu().numpy() for t in args]

    def answers(of):
        logits, value = [t.detach().cpu().numpy() for t in learner.heads(learner.features(*args))]
        got, v = of.infer_gomoku(*host, api.OUT_LOGITS)
        # the same tower and the same fp32 heads in another order of additions: pc * S * S terms a logit
        assert np.abs(got - logits).max() <= 1e-4 * (1 + np.abs(logits).max()) and np.abs(v - value).max() <= 1e-4
        return logits
    before = answers(net)
    loss, value_loss, stats, norm = learner.step_search(*args, b["visits"], b["outcome"], b["legal_bits"], lr=1e-2)
    lp = torch.log_softmax(torch.from_numpy(before).double().masked_fill(~torch.from_numpy(legal), -float("inf")), 1)
    t = b["visits"].double().cpu() * torch.from_numpy(legal)
    want = -(t * lp.masked_fill(t == 0, 0)).sum(1) / t.sum(1)
    assert np.abs(stats[:, 0].double().cpu().numpy() - want.numpy()).max() <= 1e-5 * (1 + float(want.abs().max()))
    after = answers(handle(learner.weights()))
    assert np.abs(after - before).max() > 1e-3
