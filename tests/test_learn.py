"""Host side of the learner, on CPU: positions and batches from self-play records."""
import numpy as np

from omoknuni_small_b200 import learn


def test_positions_and_batch():
    pi = np.zeros(25, np.float32)
    pi[3] = 1
    rec = {"winner": 2, "moves": [4, 7], "opening": [0, 24], "policies": [pi.tolist(), pi.tolist()]}
    ps = list(learn.positions_of(rec))
    assert [p[0] for p in ps] == [[0, 24], [0, 24, 4]] and [p[2] for p in ps] == [-1.0, 1.0]
    b = learn.batch_of(ps, 5)
    assert b["history"][1, :4].tolist() == [4, 24, 0, -1] and b["n_hist"].tolist() == [2, 3] and b["to_move"].tolist() == [1, 2]
    legal = np.unpackbits(b["legal_bits"].view(np.uint8), bitorder="little").reshape(2, 32)
    assert legal[0].sum() == 23 and not legal[0, [0, 24]].any() and not legal[1, [0, 24, 4]].any() and not legal[:, 25:].any()
    assert b["target"][0, 3] == 1 and b["outcome"].tolist() == [-1.0, 1.0]
    # a drawn game; more moves than a history holds
    rec = {"winner": 0, "moves": list(range(20)), "policies": [pi.tolist()] * 20}
    ps = list(learn.positions_of(rec))
    assert all(p[2] == 0 for p in ps)
    b = learn.batch_of(ps[-1:], 5)
    assert b["history"][0].tolist() == list(range(18, 2, -1)) and b["n_hist"][0] == 16 and b["to_move"][0] == 2
