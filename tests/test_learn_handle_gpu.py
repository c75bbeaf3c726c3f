"""A learner's steps between the answers and searches of the handle it was given: nothing reads or writes the handle's
activations out of turn, on whatever stream and from whatever thread."""
import threading

import numpy as np
import pytest

from omoknuni_small_b200 import synth
from test_learn_gpu import batch, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


def test_answers_and_searches_between_steps(api):
    import torch
    net, _, learner = make(api, B=256)
    b, _ = batch(250)
    args = (b["history"], b["n_hist"], b["to_move"])
    _, hist, nh, tm = synth.make_gomoku_games(200, 15, seed=7)
    games = [[i, 30 + i] for i in range(8)]

    def search():
        return api.Search(net, n_trees=8, sims_per_move=64, leaf_batch=64, max_depth=16, seed=5).run(games)[0]
    want_x = learner.features(*args)
    torch.cuda.synchronize()
    want_p, want_v = net.infer_gomoku(hist, nh, tm, api.OUT_LOGITS)
    want_pi = search()
    heavy = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    streams = [torch.cuda.current_stream(), torch.cuda.Stream()]
    for turn in range(8):
        with torch.cuda.stream(streams[turn % 2]):
            if turn < 4:
                for _ in range(10):
                    torch.mm(heavy, heavy)           # milliseconds of work ahead of the tower
            x = learner.features(*args)
            if turn % 4 < 2:
                p, v = net.infer_gomoku(hist, nh, tm, api.OUT_LOGITS)
                y = learner.features(*args)          # at once behind the answer, whose stream is the handle's
                pi = search()
            else:
                pi = search()
                y = learner.features(*args)
                p, v = net.infer_gomoku(hist, nh, tm, api.OUT_LOGITS)
            torch.cuda.synchronize()
        assert torch.equal(x, want_x) and torch.equal(y, want_x)
        assert np.array_equal(p, want_p) and np.array_equal(v, want_v) and np.array_equal(pi, want_pi)


def test_steps_while_another_thread_searches_and_answers(api):
    import torch
    net, _, learner = make(api, B=256)
    b, _ = batch(250)
    args = (b["history"], b["n_hist"], b["to_move"])
    _, hist, nh, tm = synth.make_gomoku_games(200, 15, seed=7)
    want_x = learner.features(*args)
    torch.cuda.synchronize()
    want_p, _ = net.infer_gomoku(hist, nh, tm, api.OUT_LOGITS)
    games = [[i, 30 + i] for i in range(8)]
    want_pi = api.Search(net, n_trees=8, sims_per_move=64, leaf_batch=64, max_depth=16, seed=5).run(games)[0]
    wrong = []

    def searches():
        for _ in range(10):
            s = api.Search(net, n_trees=8, sims_per_move=64, leaf_batch=64, max_depth=16, seed=5)
            if not np.array_equal(s.run(games)[0], want_pi):
                wrong.append("search")

    def answers():
        for _ in range(30):
            if not np.array_equal(net.infer_gomoku(hist, nh, tm, api.OUT_LOGITS)[0], want_p):
                wrong.append("answer")
    threads = [threading.Thread(target=f) for f in (searches, answers)]
    for t in threads:
        t.start()
    got = [learner.features(*args) for _ in range(30)]
    for t in threads:
        t.join(timeout=120)
    torch.cuda.synchronize()
    assert not wrong and all(torch.equal(x, want_x) for x in got)


def test_copied_tower_output(api):
    """A board tensor as the handle's own, with zeros behind its boards though a larger batch went before; no captures."""
    import torch
    net, _, learner = make(api, B=64)
    _, hist, nh, tm = synth.make_gomoku_games(64, 15, seed=7)
    net.infer_gomoku(hist, nh, tm)
    b, _ = batch(5)
    planes = api.encode_gomoku(b["history"], b["n_hist"], b["to_move"], 15, 17, 64)
    got = net.tower_copy_device(planes, 5)
    torch.cuda.synchronize()
    raw = np.zeros(5 * 256 * 64 + 32 * 64, np.int16)
    api.check(api.lib().ob200_copy_to_host(raw.ctypes.data, net.tower_output_ptr(), raw.nbytes))
    assert np.array_equal(got[:raw.size].cpu().numpy(), raw) and not got[raw.size:].any() and raw.any()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        planes.add_(0)
        with pytest.raises(api.Error):
            net.tower_copy_device(planes, 5, got)
    with pytest.raises(api.Error):
        net.tower_copy_device(torch.zeros_like(planes), 0, got[:0].new_zeros(64 * 64))
