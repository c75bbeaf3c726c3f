"""Sizes and placements that the policy losses refuse, without a device."""
import pytest

from test_train_refusals import clipped, rows, search


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


def test_matrices_beyond_any_memory(api):
    """Offsets in bytes would leave 64 bits, and with them the check of what overlaps: 2^31 rows of 2^31 elements."""
    n, most = (1 << 31) - 1, 1 << 31
    for far in (dict(logits_pitch=most), dict(grad_pitch=most), dict(logits_pitch=most, grad_pitch=most)):
        assert search(api, rows(api, n=n, **far)) == clipped(api, rows(api, n=n, **far)) == api.ERR_INVALID
    assert search(api, rows(api, n=n), pitch=most) == api.ERR_INVALID
    assert clipped(api, rows(api, n=n), ref=0x4000000, pitch=most, kl=0.1) == api.ERR_INVALID
    assert search(api, rows(api, n=n, legal_bits=0x5000, mask_words=n)) == api.ERR_INVALID
    # the gradient of the last row on the logits: an offset of 2^64 bytes, 0 in 64 bits
    r = rows(api, n=n, n_actions=225, logits_pitch=most, grad_pitch=most, grad=0x10000 + 64)
    assert search(api, r) == api.ERR_INVALID


PLACES = dict(logits=0x10000, grad=0x900000, loss=0x20000, stats=0x30000, row_weight=0x40000, legal_bits=0x50000)
BYTES = dict(logits=225 * 32, grad=225 * 32, target=225 * 32, ref=225 * 32, loss=32, stats=128, row_weight=32, legal_bits=256, act=32, old=32, adv=32)


def calls(api, name, at):
    """Both losses with `name` at another place, where they have it."""
    full = dict(PLACES, mask_words=8, **({name: at} if name in PLACES else {}))
    out = []
    if name not in ("act", "old", "adv", "ref"):
        out.append(search(api, rows(api, **full), **({"target": at} if name == "target" else {})))
    if name != "target":
        kw = dict(act=0x3000000, old=0x3001000, adv=0x3002000, ref=0x4000000, pitch=225, kl=0.1)
        if name in kw:
            kw[name] = at
        out.append(clipped(api, rows(api, **full), **kw))
    return out


def place_of(name):
    return dict(PLACES, target=0x2000000, ref=0x4000000, act=0x3000000, old=0x3001000, adv=0x3002000)[name]


@pytest.mark.parametrize("other", sorted(BYTES))
@pytest.mark.parametrize("written", ["loss", "stats", "grad"])
def test_outputs_on_other_memory(api, written, other):
    """At the same place, at its last bytes, ending in its first: what a call writes shares no byte with anything else it has."""
    if written == other or (written, other) == ("grad", "logits"):
        pytest.skip("the same, or allowed")
    step = 16                                    # keeps every pointer aligned
    for at in (place_of(other), place_of(other) + BYTES[other] - step, place_of(other) - BYTES[written] + step):
        mine = place_of(written)
        # the other one is moved, so that the losses that have it are called
        shift = mine - (at - place_of(other)) if other not in PLACES else None
        got = calls(api, other, shift) if shift is not None else calls(api, written, at)
        assert got and all(rc == api.ERR_INVALID for rc in got), (hex(at), got)


def test_outputs_between_rows_are_allowed(api):
    """loss in the columns that lie between the rows of a wider matrix, and everything apart."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a device: the pointers are made up")
    assert calls(api, "loss", PLACES["loss"]) == [2, 2]
    for at, want in ((0x10000 + 225 * 4, 2), (0x10000 + 225 * 4 + 28, 2), (0x10000 + 240 * 4 - 28, 1), (0x10000 + 225 * 4 - 4, 1)):
        r = rows(api, logits_pitch=240, loss=at, n=8)
        assert search(api, r) == (want if want == 2 else api.ERR_INVALID), hex(at)
