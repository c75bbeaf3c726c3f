"""What a learner refuses of its positions, on CPU."""
import pytest


def test_positions_refused():
    import torch
    from omoknuni_small_b200 import capi, learn
    cpu = torch.device("cpu")

    def args(**kw):
        good = dict(history=torch.zeros((5, 16), dtype=torch.int16), n_hist=torch.zeros(5, dtype=torch.uint8),
                    to_move=torch.ones(5, dtype=torch.uint8), outcome=torch.zeros(5))
        return dict(good, **kw)
    learn.check_positions(cpu, **args())
    learn.check_positions(cpu, **args(outcome=None))
    learn.check_positions(cpu, **args(outcome=torch.zeros(5, dtype=torch.int64)))
    for kw in (dict(history=torch.zeros((5, 16), dtype=torch.int32)), dict(history=torch.zeros((5, 15), dtype=torch.int16)),
               dict(history=torch.zeros(80, dtype=torch.int16)), dict(history=torch.zeros((5, 32), dtype=torch.int16)[:, ::2]),
               dict(history=torch.tensor(0, dtype=torch.int16)), dict(n_hist=torch.zeros(4, dtype=torch.uint8)),
               dict(n_hist=torch.zeros(5, dtype=torch.int64)), dict(to_move=torch.ones((5, 1), dtype=torch.uint8)),
               dict(to_move=torch.ones(10, dtype=torch.uint8)[::2]), dict(outcome=torch.zeros((5, 1))), dict(outcome=torch.zeros(4)),
               dict(n_hist=torch.zeros(5, dtype=torch.uint8, device="meta"))):
        with pytest.raises(capi.Error) as e:
            learn.check_positions(cpu, **args(**kw))
        assert e.value.code == capi.ERR_INVALID
