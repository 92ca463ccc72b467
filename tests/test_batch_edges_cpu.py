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


@pytest.mark.parametrize("where", [
    dict(out=P + 16), dict(out=P - 16), dict(out=P, x_dtype=0), dict(out=P, qs=1024),  # q shifted, of another type, with gaps
    dict(out=2 * P), dict(out=2 * P + 256), dict(out=3 * P - 3 * 1024 + 16), dict(out=P, k=P + 2048)])
def test_append_refuses_overlapping_q_out(L, where):
    from q4b import _lib
    a = dict(out=4 * P, k=2 * P, v=3 * P, x_dtype=1, qs=512)
    a.update(where)
    b = _lib.Batch(q_start=5 * P, seq_lens=5 * P, page_table=5 * P, batch=2, table_width=4, table_stride=4, prefix_len=0)
    c = _lib.PagedKV(k=6 * P, v=7 * P, dtype=_lib.F16, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, page_stride=2048,
                     slot_stride=128, head_stride=64)
    rc = L.q4b_paged_rope_append(P, a["k"], a["v"], a["x_dtype"], a["qs"], 128, 128, 3, 8, 8 * P, 9 * P, 32, 64, 64, 0,
                                 ctypes.byref(b), ctypes.byref(c), a["out"], None)
    assert rc == _lib.Q4B_EINVAL and b"overlap" in L.q4b_last_error()
