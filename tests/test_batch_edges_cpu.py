"""Refusals of the batched serving operators' C ABI that the device never sees (no GPU needed)."""

import ctypes

import pytest

P = 1 << 20  # never dereferenced: the check comes before any launch


@pytest.fixture(scope="module")
def L():
    from q4b import _lib
    return _lib.lib()


@pytest.mark.parametrize("where", [
    dict(out=P), dict(out=P + 4), dict(out=P + 12), dict(out=P - 12),  # tokens: the same, shifted by one, at either end
    dict(out=2 * P), dict(accepted=P + 4), dict(accepted=2 * P + 12), dict(out=3 * P), dict(out=3 * P + 8),
    dict(accepted=3 * P + 8), dict(out=4 * P, accepted=4 * P + 12)])
def test_verify_refuses_overlapping_results(L, where):
    """Results over inputs would be read by other CTAs of the step while they are written."""
    from q4b import _lib
    a = dict(out=4 * P, accepted=5 * P)
    a.update(where)
    rc = L.q4b_verify_drafts(6 * P, None, 0, 100, 100, 100, P, 2 * P, 4, 3 * P, 2, a["out"], a["accepted"], None)
    assert rc == _lib.Q4B_EINVAL and b"overlap" in L.q4b_last_error()
