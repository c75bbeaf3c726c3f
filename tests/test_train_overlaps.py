"""Memory that a call of the training operators writes and that is somebody else's too: refused, without a device."""
import ctypes as C

import pytest

from test_train_refusals import config, tensors


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


def adamw(api, t, n, bits):
    return api.lib().ob200_launch_adamw(t, n, C.byref(config(api, state_bits=bits)), None)


def allowed(rc):
    """No argument error: without a device the device check answers, with one there is no call to try."""
    return rc == 2


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("order", ["memory", "shuffled"])
def test_adamw_memory_that_is_written_twice(api, bits, order):
    es = 4 if bits == 32 else 1
    size = 1000 * es
    fields = ["param", "exp_avg", "exp_avg_sq"] + (["exp_avg_scale", "exp_avg_sq_scale"] if bits == 8 else [])
    bytes_of = dict(param=4000, exp_avg=size, exp_avg_sq=size, exp_avg_scale=16, exp_avg_sq_scale=16)

    def three():
        t = tensors(api, 3)
        if order == "shuffled":
            t[0], t[2] = api.TrainTensor.from_buffer_copy(t[2]), api.TrainTensor.from_buffer_copy(t[0])
        return t
    for i in range(3):
        for j in range(3):
            for a in fields:
                for b in fields:
                    if (i, a) == (j, b):
                        continue
                    for shift in (0, bytes_of[b] - 4, 4 - bytes_of[a]):       # the same place, its last four bytes, its first four
                        t = three()
                        setattr(t[i], a, getattr(t[j], b) + shift)
                        assert adamw(api, t, 3, bits) == api.ERR_INVALID, (i, a, j, b, shift)
    import torch
    if torch.cuda.is_available():
        pytest.skip("the pointers are made up: calls without a mistake are tried on a machine without a device")
    assert allowed(adamw(api, three(), 3, bits))
    t = three()                                  # end to end, every kind, is apart
    at = 0x100000
    for i in (2, 0, 1):
        for f in fields:
            setattr(t[i], f, at)
            at += bytes_of[f]
    assert allowed(adamw(api, t, 3, bits))
    for e in t:                                  # without elements nothing is written
        e.numel, e.param = 0, 0x100000
    assert allowed(adamw(api, t, 3, bits))
    if bits == 32:                               # scales are no memory of such a call
        t = three()
        t[0].exp_avg_scale = t[1].param
        assert allowed(adamw(api, t, 3, bits))


def test_eps_that_is_subnormal(api):
    """Its reciprocal would be infinite where a second moment is 0, and the weight beside a zero gradient NaN."""
    for eps in (1e-38, 1e-40, 2.0 ** -149):
        assert api.lib().ob200_launch_adamw(tensors(api), 2, C.byref(config(api, eps=eps)), None) == api.ERR_INVALID
