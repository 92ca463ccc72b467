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


def _attend_batch(lib, **kw):
    d = dict(q_start=P, seq_lens=P, page_table=P, batch=32, table_width=32, table_stride=8192, prefix_len=2048)
    d.update(kw)
    kv = dict(k=P, v=P, dtype=lib.F16, n_pages=10_000, page_size=16, n_kv_heads=8, head_dim=128, page_stride=16 * 8 * 128,
              slot_stride=8 * 128, head_stride=128)
    return lib.Batch(**d), lib.PagedKV(**kv)


def test_attention_plans_by_told_lengths_not_by_the_tables_width(L):
    """The workspace's size shows how the kernels share the SMs: the same for a table of any width if own_keys is told."""
    from q4b import _lib
    size = lambda **kw: L.q4b_prefix_attention_workspace(32, 24, *map(ctypes.byref, _attend_batch(_lib, **kw)))  # noqa: E731
    told = {size(own_keys=300, table_width=w) for w in (32, 128, 512, 8192)}
    assert len(told) == 1 and told != {0}
    assert size(table_width=32) != size(table_width=8192)  # the width is all that is known then
    # a prompt chunk among idle sequences: the own keys of many rows need places of the tensor-core kernel
    assert size(prefix_len=0, max_new=20) > size(prefix_len=0)


@pytest.mark.parametrize("bad", [dict(max_new=-1), dict(own_keys=-1)])
def test_attention_refuses_negative_hints(L, bad):
    from q4b import _lib
    b, kv = _attend_batch(_lib, **bad)
    assert L.q4b_prefix_attention_workspace(32, 24, ctypes.byref(b), ctypes.byref(kv)) == 0
    assert b"negative" in L.q4b_last_error()
