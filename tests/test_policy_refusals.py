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
