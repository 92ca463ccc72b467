"""CPU-side refusals of the batched serving operators: bad arguments are reported on the host before any launch
(no GPU needed), by the Python wrappers and by the C ABI."""

import ctypes

import numpy as np
import pytest
import torch

import batch_ref as R


@pytest.fixture(scope="module")
def L():
    from q4b import _lib
    return _lib.lib()


def _batch(lib, **kw):
    d = dict(q_start=16, seq_lens=16, page_table=16, batch=2, table_width=4, table_stride=4, prefix_len=0)
    d.update(kw)
    return lib.Batch(**d)


def _kv(lib, **kw):
    d = dict(k=16, v=16, dtype=lib.F16, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, page_stride=2048,
             slot_stride=128, head_stride=64)
    d.update(kw)
    return lib.PagedKV(**d)


APPEND_BAD = [
    (dict(q=None), {}, {}, b"null"),
    (dict(x_dtype=2), {}, {}, b"type"),
    (dict(x_dtype=9), {}, {}, b"type"),
    (dict(rot=24), {}, {}, b"multiples of 16"),
    (dict(rot=80), {}, {}, b"rot_dim"),
    (dict(cos=None), {}, {}, b"tables"),
    (dict(qs=129), {}, {}, b"strides"),
    (dict(q=24), {}, {}, b"aligned"),
    (dict(rows=-1), {}, {}, b"negative"),
    (dict(heads=0), {}, {}, b"n_heads"),
    ({}, dict(q_start=None), {}, b"null"),
    ({}, dict(seq_lens=None), {}, b"null"),
    ({}, dict(prefix_len=-1), {}, b"negative"),
    ({}, dict(table_stride=3), {}, b"overlap"),
    ({}, {}, dict(dtype=0), b"fp16 or bf16"),
    ({}, {}, dict(head_dim=40), b"multiples of 16"),
    ({}, {}, dict(slot_stride=68), b"strides"),
    ({}, {}, dict(k=8), b"aligned"),
    ({}, {}, dict(n_pages=0), b"empty"),
    ({}, {}, dict(slot_stride=0), b"overlap"),
    ({}, {}, dict(page_stride=0), b"overlap"),
]


@pytest.mark.parametrize("args,batch,kv,word", APPEND_BAD)
def test_append_refuses(L, args, batch, kv, word):
    from q4b import _lib
    a = dict(q=16, k=16, v=16, x_dtype=1, qs=512, ks=128, vs=128, rows=3, heads=8, cos=16, sin=16, ts=32, tr=64,
             rot=64, out=16)
    a.update(args)
    b, c = _batch(_lib, **batch), _kv(_lib, **kv)
    rc = L.q4b_paged_rope_append(a["q"], a["k"], a["v"], a["x_dtype"], a["qs"], a["ks"], a["vs"], a["rows"],
                                 a["heads"], a["cos"], a["sin"], a["ts"], a["tr"], a["rot"], 0, ctypes.byref(b),
                                 ctypes.byref(c), a["out"], None)
    assert rc == _lib.Q4B_EINVAL
    assert word in L.q4b_last_error(), L.q4b_last_error()


ATTEND_BAD = [
    (dict(q=None), {}, {}, b"null"), (dict(out=None), {}, {}, b"null"),
    (dict(pages=None), dict(prefix_len=5), {}, b"null"), (dict(qs=511), {}, {}, b"even strides"),
    (dict(q=18), {}, {}, b"aligned"), (dict(out=8), {}, {}, b"aligned"), (dict(scale=0.0), {}, {}, b"scale"),
    (dict(scale=float("nan")), {}, {}, b"scale"), (dict(scale=float("inf")), {}, {}, b"scale"),
    (dict(ws=None), {}, {}, b"workspace"), (dict(ws=4096 + 16), {}, {}, b"workspace"), (dict(wsb=-1), {}, {}, b"workspace"),
    (dict(heads=3), {}, {}, b"n_kv_heads"), (dict(heads=0), {}, {}, b"n_kv_heads"), (dict(rows=-1), {}, {}, b"negative"),
    ({}, dict(batch=-1), {}, b"negative"), ({}, dict(q_start=None), {}, b"null"),
    ({}, dict(prefix_len=2**31 - 1), {}, b"prefix_len"), ({}, {}, dict(dtype=7), b"fp16 or bf16"), ({}, {}, dict(v=24), b"aligned"),
    ({}, {}, dict(page_stride=-8), b"strides"),
]


@pytest.mark.parametrize("args,batch,kv,word", ATTEND_BAD)
def test_attention_refuses(L, args, batch, kv, word):
    from q4b import _lib
    a = dict(q=16, qs=512, hs=64, rows=3, heads=8, scale=0.125, pages=16, out=16, ws=4096, wsb=0)
    a.update(args)
    b, c = _batch(_lib, **batch), _kv(_lib, **kv)
    need = L.q4b_prefix_attention_workspace(a["rows"], a["heads"], ctypes.byref(b), ctypes.byref(c))
    rc = L.q4b_prefix_attention(a["q"], a["qs"], a["hs"], a["rows"], a["heads"], a["scale"], a["pages"],
                                ctypes.byref(b), ctypes.byref(c), a["out"], a["ws"], max(need + a["wsb"], 0), None)
    assert rc == _lib.Q4B_EINVAL
    assert word in L.q4b_last_error(), L.q4b_last_error()


@pytest.mark.parametrize("rows,batch,kv", [(3, {}, dict(head_dim=48)), (3, dict(batch=5000), {}),
                                           (20_000_000, {}, {}), (3, dict(table_width=2**30, table_stride=2**30), dict(page_size=64))])
def test_attention_names_what_it_does_not_handle(L, rows, batch, kv):
    """Valid calls beyond the kernels' bounds: no workspace size, and an error of their own."""
    from q4b import _lib
    b, c = _batch(_lib, **batch), _kv(_lib, **kv)
    assert L.q4b_prefix_attention_workspace(rows, 8, ctypes.byref(b), ctypes.byref(c)) == 0
    rc = L.q4b_prefix_attention(16, 512, 64, rows, 8, 0.125, 16, ctypes.byref(b), ctypes.byref(c), 16, 4096, 1 << 40, None)
    assert rc == _lib.Q4B_EUNSUPPORTED


VERIFY_BAD = [
    (dict(target=None), b"null"), (dict(tokens=None), b"null"), (dict(q_start=None), b"null"),
    (dict(accepted=None), b"null"), (dict(dtype=3), b"fp32"), (dict(vocab=0), b"vocab"),
    (dict(vocab=(1 << 20) + 1), b"vocab"), (dict(ts=99), b"overlap"), (dict(ds=99), b"overlap"),
    (dict(rows=-1), b"negative"), (dict(batch=-1), b"negative"), (dict(target=18), b"misaligned"),
]


@pytest.mark.parametrize("args,word", VERIFY_BAD)
def test_verify_refuses(L, args, word):
    from q4b import _lib
    a = dict(target=16, draft=16, dtype=0, ts=100, ds=100, vocab=100, tokens=16, uniforms=16, rows=4, q_start=16,
             batch=2, out=16, accepted=16)
    a.update(args)
    rc = L.q4b_verify_drafts(a["target"], a["draft"], a["dtype"], a["ts"], a["ds"], a["vocab"], a["tokens"],
                             a["uniforms"], a["rows"], a["q_start"], a["batch"], a["out"], a["accepted"], None)
    assert rc == _lib.Q4B_EINVAL
    assert word in L.q4b_last_error(), L.q4b_last_error()


def test_wrappers_refuse_cpu_tensors():
    import q4b
    t = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 16)
    p = torch.zeros(1, 16, 1, 16, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        q4b.paged_rope_append(x, x, x, p, p, t[None], t, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        q4b.prefix_attention(x, p, p, t, 0, t[None], t, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        q4b.verify_drafts(torch.zeros(1, 8), None, t, torch.zeros(1), torch.zeros(2, dtype=torch.int32))


def test_empty_calls_launch_nothing(L):
    from q4b import _lib
    b, c = _batch(_lib, batch=0), _kv(_lib)
    assert L.q4b_paged_rope_append(16, 16, 16, 1, 512, 128, 128, 3, 8, 16, 16, 32, 64, 64, 0, ctypes.byref(b),
                                   ctypes.byref(c), 16, None) == 0
    assert L.q4b_verify_drafts(16, 16, 0, 100, 100, 100, 16, 16, 4, 16, 0, 16, 16, None) == 0
    assert L.q4b_prefix_attention(16, 512, 64, 3, 8, 0.125, None, ctypes.byref(b), ctypes.byref(c), 16, None, 0, None) == 0


def test_plain_forms_agree_with_hand_made_values():
    """The oracle itself, on values that can be worked out by hand."""
    p = np.array([[0.5, 0.5, 0.0], [0.1, 0.2, 0.7]])
    d = np.array([[0.0, 0.5, 0.5], [0.3, 0.3, 0.4]])
    # draft 1: 0.9 * 0.5 < 0.5 kept; the last row draws: cumsum 0.1, 0.3, 1.0 against 0.25
    out, acc = R.verify(p, d, np.array([0, 1]), np.array([0.9, 0.25]), [0, 2])
    assert out == [1, 1] and acc == [1]
    # draft 2 has no target probability: rejected; the residual is (0.5, 0, 0)
    out, acc = R.verify(p, d, np.array([0, 2]), np.array([0.0, 0.99]), [0, 2])
    assert out == [0, -1] and acc == [0]
    x = R.rotate(np.array([[1.0, 0.0, 5.0]]), np.array([0.6]), np.array([0.8]), "half")
    assert x.tolist() == [[0.6, 0.8, 5.0]]
    kp = np.zeros((2, 2, 1, 2))
    kp[1, 0, 0] = [1.0, 0.0]
    vp = np.ones((2, 2, 1, 2)) * np.arange(1, 3)[:, None, None, None]
    b = R.make_batch([(1, 2)], 2, 2)
    b["page_table"][0, 0] = 1
    out = R.attention(np.array([[[2.0, 0.0]]]), kp, vp, b, 2, scale=1.0)
    assert np.allclose(out, 2.0)
