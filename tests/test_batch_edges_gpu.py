"""Edges of the batched serving operators: contents, lengths, aliases and plans that the parity tests do not reach."""

import numpy as np
import pytest
import torch

import batch_ref as R
from test_batch_gpu import (DEV, _append_case, _attend_case, _check_attend, _close_rounded, _dev, _f64, _run_append,  # noqa: F401
                            _run_attend, _verify_case, q4b)

pytestmark = pytest.mark.gpu


# ---- prefix_attention: what stands behind the last key ------------------------------------------------


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,g,page", [(1, 3, 16), (1, 8, 64), (3, 5, 8), (2, 8, 24), (20, 4, 16), (30, 8, 64)])
def test_rest_of_a_page_never_shows(q4b, hd, new, g, page):  # noqa: F811
    """Own keys that end at every place of a 64-key (and of a 128-key) tile, NaN keys and infinite values behind them, in
    the narrow kernel (few rows a sequence) and the tensor-core one (more than 64 rows x heads), again and again over the
    same shared memory."""
    lens = [(new, max(n, new)) for n in range(1, 131)]
    case = _attend_case(lens, page, 0, 2 * g, 2, hd, torch.float16, seed=page + g)
    out, _, live = _run_attend(q4b, case, page)
    assert live.all() and bool(torch.isfinite(out).all())


# ---- prefix_attention: waits that give up ---------------------------------------------------------------


@pytest.mark.parametrize("lens,prefix,H,Hkv,hd", [
    ([(1, 700), (1, 90), (2, 33)] * 9, 0, 8, 2, 128),  # the narrow kernel
    ([(1, 5)] * 150, 4500, 8, 4, 64),  # both, a few tiles each
    ([(1, 1900)] * 40 + [(90, 2000)], 9000, 8, 2, 128),  # both, rings that go round, own keys on the tensor cores too
])
def test_waits_that_give_up_are_reported(q4b, lens, prefix, H, Hkv, hd):  # noqa: F811
    """With a limit of zero every wait gives up: each row that has keys is NaN, none is stale, the status tells, and the next
    call is right again. The waits end by themselves; nothing is left out or broken for it."""
    L = q4b.lib()
    case = _attend_case(lens, 16, prefix, H, Hkv, hd, torch.float16, seed=3)
    b, q, kp, vp = case
    d = _dev(b)
    call = lambda: q4b.prefix_attention(q, kp, vp, d["prefix_pages"], prefix, d["page_table"], d["seq_lens"], d["q_start"])  # noqa: E731
    assert L.q4b_device_status(1) == 0
    L.q4b_prefix_attention_wait_limit(0)
    try:
        outs = [call() for _ in range(3)]
        torch.cuda.synchronize()
    finally:
        L.q4b_prefix_attention_wait_limit(10**9)
    for o in outs:
        assert bool(torch.isnan(o).all())
    assert L.q4b_device_status(1) == -3 and L.q4b_device_status(1) == 0
    _run_attend(q4b, case, 16)
    assert L.q4b_device_status(1) == 0


# ---- paged_rope_append: sequences that outgrow their tables ---------------------------------------------


@pytest.mark.parametrize("lens,width", [
    ([(1, 33), (1, 32), (2, 20)], 4),  # one token behind the last slot; the last slot; inside
    ([(4, 34), (3, 50), (40, 45)], 4),  # rows on both sides of the table's end, all behind it, a chunk across it
    ([(2, 2), (1, 9)], 0),  # no pages at all
    ([(3, -5), (2, 1), (1, 0)], 4),  # negative, and shorter than the new rows
])
@pytest.mark.parametrize("prefix", [0, 7])
def test_append_behind_the_table_is_dropped(q4b, lens, width, prefix):  # noqa: F811
    """A row keeps its position whatever the table holds: it is rotated there, and written nowhere else."""
    page, H, Hkv, hd = 8, 4, 2, 64
    rng = np.random.default_rng(len(lens) + width)
    b = dict(q_start=np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32), prefix_len=prefix,
             seq_lens=np.array([o for _, o in lens], dtype=np.int32),
             page_table=rng.permutation(20)[:len(lens) * width].reshape(len(lens), width).astype(np.int32),
             prefix_pages=np.zeros(0, dtype=np.int32), rows=sum(n for n, _ in lens))
    g = torch.Generator(device=DEV).manual_seed(width)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    q, k, v = rn(b["rows"], H, hd), rn(b["rows"], Hkv, hd), rn(b["rows"], Hkv, hd)
    kp, vp = (rn(20, page, Hkv, hd).half() for _ in range(2))
    ang = torch.arange(100, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(hd // 2, dtype=torch.float64) / (hd // 2))
    _run_append(q4b, (b, q, k, v, kp, vp, ang.cos().float().to(DEV), ang.sin().float().to(DEV)), "half", page, "float16")


# ---- prefix_attention: the same lengths -----------------------------------------------------------------


@pytest.mark.parametrize("lens,width,prefix,H,Hkv,hd,page", [
    ([(1, 33), (4, 34), (3, 50), (2, 20)], 4, 0, 8, 2, 64, 8),
    ([(1, 33), (4, 34), (3, 50), (2, 20)], 4, 21, 8, 2, 32, 20),  # the wide kernel
    ([(40, 70), (100, 300), (3, 2**31 - 1)], 4, 100, 4, 2, 128, 16),  # the tensor cores: rows across the table's end
    ([(2, 2), (1, 9)], 0, 5, 2, 2, 128, 16),
    ([(70, -3), (3, -2**31), (2, 1)], 3, 0, 4, 2, 64, 16),
    ([(1, 40)] * 150, 2, 4500, 8, 4, 64, 16),
])
def test_attend_keys_behind_the_table(q4b, lens, width, prefix, H, Hkv, hd, page):  # noqa: F811
    """Row j sees the own keys 0 .. seq_lens - n + j that the table holds, whatever seq_lens is."""
    rng = np.random.default_rng(width)
    pages = len(lens) * width + -(-prefix // page) + 1
    ids = rng.permutation(pages).astype(np.int32)
    rows = sum(n for n, _ in lens)
    g = torch.Generator(device=DEV).manual_seed(width)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).half()  # noqa: E731
    q, kp, vp = rn(rows, H, hd), rn(pages, page, Hkv, hd), rn(pages, page, Hkv, hd)
    b = dict(q_start=np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32), prefix_len=prefix, rows=rows,
             seq_lens=np.array([o for _, o in lens], dtype=np.int32),
             page_table=ids[:len(lens) * width].reshape(len(lens), width), prefix_pages=ids[len(lens) * width:pages - 1])
    d = _dev(b)
    got = _f64(q4b.prefix_attention(q, kp, vp, d["prefix_pages"], prefix, d["page_table"], d["seq_lens"], d["q_start"]))
    # the 64-bit form counts keys up to seq_lens: columns without a page behind the table, up to where the last row looks
    far = width * page + rows + 1
    wide = np.concatenate([b["page_table"], np.full((len(lens), -(-far // page) - width), -1, dtype=np.int32)], 1)
    long = np.minimum(b["seq_lens"], far)  # beyond this every row sees all that the table holds
    ref = R.attention(_f64(q), _f64(kp), _f64(vp), dict(b, page_table=wide, seq_lens=np.maximum(long, 0)), page)
    _check_attend(got.reshape(ref.shape), ref, _f64(vp), torch.float16, np.ones(rows, dtype=bool))


# ---- verify_drafts: sums of many values -----------------------------------------------------------------


@pytest.mark.parametrize("drafts,batch", [(False, 190), (True, 150)])
def test_verify_sums_do_not_drift(q4b, drafts, batch):  # noqa: F811
    """The largest vocabulary with few CTAs a sequence: 256 large weights in the first half, equal ones of 2^-24.3 of
    those everywhere, half of the mass at the very end. All weights are whole multiples of 2^-48, so that the running
    sums are exact in 64-bit integers; the numbers lie so that the marks fall between the two, at least 2^-38 of the sum away
    from the next border."""
    V, unit = 1 << 20, 2.0**-48
    per = 2 if drafts else 1
    target = torch.zeros(batch * per, V, device=DEV)
    draft = torch.zeros(batch * per, V, device=DEV) if drafts else None
    uniforms = torch.zeros(batch * per)
    want = []
    rng = np.random.default_rng(5)
    for b in range(batch):
        w = torch.full((V,), 54613 + 8 * b, dtype=torch.int64, device=DEV)
        w.view(16, -1)[:8, :128:4] = 1 << 40
        w[-1] = 1 << 48
        p = w.clone()
        if drafts:  # p - d is w; the draft 5 has no target probability
            w[5] = p[5] = 0
            d = torch.where(w < 1 << 20, 1 << 16, 0)
            p = p + d
            p[5], d[5] = 0, 1 << 16
            draft[b * per] = (d.double() * unit).float()
        target[b * per] = (p.double() * unit).float()
        acc = torch.cumsum(w, 0).cpu().numpy()
        total = int(acc[-1])
        while True:
            k = int(int(acc[rng.integers(V // 2 + 1000, V - 1000)]) * 2**24 / total)
            mark = k * total >> 24
            j = int(np.searchsorted(acc, mark, side="right"))
            if min(mark - int(acc[j - 1]), int(acc[j]) - mark) > total >> 38 and V // 2 < j < V - 1:
                break
        uniforms[b * per + per - 1] = k / 2**24
        want.append(j)
    tokens = torch.full((batch * per,), 5, dtype=torch.int32, device=DEV)
    q_start = torch.arange(0, batch * per + 1, per, dtype=torch.int32, device=DEV)
    got, acc = q4b.verify_drafts(target, draft, tokens, uniforms.to(DEV), q_start)
    assert acc.tolist() == [0] * batch
    assert got.view(batch, per)[:, 0].tolist() == want


# ---- prefix_attention: many small weights beside a large one ---------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,prefix,H,Hkv,hd,page", [
    ([(1, 40000), (1, 9000)], 0, 4, 1, 128, 16),  # the narrow kernel, 8 and 16 rows
    ([(3, 40000), (2, 30000)], 0, 8, 2, 64, 16),
    ([(2, 40000)], 0, 8, 2, 64, 20),  # the wide kernel: keys shared by the warps, and rows
    ([(30, 40000)], 0, 4, 2, 32, 16),
    ([(1, 1)] * 40, 40000, 8, 2, 128, 16),  # the tensor-core kernel: the prefix, and own keys
    ([(30, 40000)], 0, 16, 2, 64, 16),
    ([(1, 20000)] * 3, 40000, 6, 3, 128, 128),  # parts of both
])
def test_small_weights_count(q4b, lens, prefix, H, Hkv, hd, page, dtype):  # noqa: F811
    """The first key has all but a thousandth of the weight, and V of zero; each of the others 2^-26 of it, and V of one. The
    result, N 2^-26 / (1 + N 2^-26) of the N others a row sees, is made of weights that fp16 cannot hold beside 1."""
    n_pages = -(-prefix // page) + sum(-(-o // page) for _, o in lens)
    b = R.make_batch(lens, page, n_pages, prefix_len=prefix)
    kp = torch.zeros(n_pages, page, Hkv, hd, dtype=dtype, device=DEV)
    vp = torch.ones_like(kp)
    for first in ([b["prefix_pages"][0]] if prefix else [t[0] for t in b["page_table"]]):
        kp[first, 0, :, 0] = 26.0
        vp[first, 0] = 0.0
    q = torch.zeros(b["rows"], H, hd, dtype=dtype, device=DEV)
    q[:, :, 0] = 1.0
    d = _dev(b)
    got = _f64(q4b.prefix_attention(q, kp, vp, d["prefix_pages"], prefix, d["page_table"], d["seq_lens"], d["q_start"],
                                    scale=float(np.log(2.0))))
    others = np.array([prefix + o - n + j for n, o in lens for j in range(n)], dtype=np.float64) * 2.0**-26
    want = np.broadcast_to((others / (1 + others))[:, None], got.shape)
    # one rounding of the result; weights are powers of two, exact in either type; exponentials and sums in fp32
    assert (np.abs(got - want) <= (torch.finfo(dtype).eps / 2 + 2.0**-15) * want).all(), np.abs(got / want - 1).max()


# ---- the torch bindings -----------------------------------------------------------------------------------


def test_out_of_memory_is_torchs(q4b):  # noqa: F811
    """A workspace or a result that does not fit raises torch.OutOfMemoryError, which a server catches to split its step."""
    b, q, kp, vp = _attend_case([(256, 256)] * 4, 16, 64, 64, 8, 128, torch.float16, 3)
    d = _dev(b)
    call = lambda **kw: q4b.prefix_attention(q, kp, vp, d["prefix_pages"], 64, d["page_table"], d["seq_lens"], d["q_start"], **kw)  # noqa: E731
    ref = call()
    big = torch.empty(1, 8, 128, dtype=torch.float16, device=DEV).expand(100_000, 8, 128)  # its result: more than torch keeps
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.0)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            call(out=ref)
        with pytest.raises(torch.OutOfMemoryError):
            q4b.paged_rope_append(big, big, big, kp, vp, d["page_table"], d["seq_lens"], d["q_start"])
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert torch.equal(call(), ref)


def test_in_place_writes_are_counted(q4b):  # noqa: F811
    """What a call writes in place has a new version, so that autograd refuses a tensor that it had saved; tensors made in
    inference mode are taken as well."""
    b, q, kp, vp = _attend_case([(2, 9), (1, 30)], 16, 20, 4, 2, 64, torch.float16, 3)
    d = _dev(b)
    meta = (d["page_table"], d["seq_lens"], d["q_start"])
    k, v = torch.randn(2, 3, 2, 64, device=DEV).half()
    leaf = torch.ones((), device=DEV, requires_grad=True)
    loss = (leaf * kp.nan_to_num(0, 0, 0)).sum() + (leaf * kp).sum()
    for out in (None, torch.empty_like(q)):
        before = (kp._version, vp._version, q._version, k._version) + (() if out is None else (out._version,))
        q4b.paged_rope_append(q, k, v, kp, vp, *meta, prefix_len=20, q_out=out)
        after = (kp._version, vp._version, q._version, k._version) + (() if out is None else (out._version,))
        assert [y - x for x, y in zip(before, after)] == [1, 1, 0, 0] + ([] if out is None else [1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    out = torch.empty(3, 256, dtype=torch.float16, device=DEV)
    version = out._version
    q4b.prefix_attention(q, kp, vp, d["prefix_pages"], 20, *meta, out=out)
    assert out._version == version + 1
    probs, toks = torch.softmax(torch.randn(3, 50, device=DEV), -1), torch.zeros(3, dtype=torch.int32, device=DEV)
    new = torch.empty(3, dtype=torch.int32, device=DEV)
    version = new._version
    q4b.verify_drafts(probs, None, toks, torch.rand(3, device=DEV), d["q_start"], out=new)
    assert new._version == version + 1
    with torch.inference_mode():
        kp2, vp2, out2 = kp.clone(), vp.clone(), torch.empty_like(out)
    q4b.paged_rope_append(q, k, v, kp2, vp2, *meta, prefix_len=20)
    assert torch.equal(q4b.prefix_attention(q, kp2, vp2, d["prefix_pages"], 20, *meta, out=out2), out)


def test_gradients_are_not_lost_silently(q4b):  # noqa: F811
    b, q, kp, vp = _attend_case([(2, 9), (1, 30)], 16, 20, 4, 2, 64, torch.float16, 3)
    d = _dev(b)
    meta = (d["page_table"], d["seq_lens"], d["q_start"])
    k = torch.randn(3, 2, 64, device=DEV).half()
    probs, toks, u = torch.softmax(torch.randn(3, 50, device=DEV), -1), torch.zeros(3, dtype=torch.int32, device=DEV), torch.rand(3, device=DEV)
    grad = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    calls = [lambda: q4b.paged_rope_append(q, grad(k), k, kp, vp, *meta, prefix_len=20),
             lambda: q4b.prefix_attention(grad(q), kp, vp, d["prefix_pages"], 20, *meta),
             lambda: q4b.verify_drafts(grad(probs), None, toks, u, d["q_start"])]
    for call in calls:
        with pytest.raises(ValueError, match="requires grad"):
            call()
        with torch.no_grad():
            call()
    ref = q4b.prefix_attention(q, kp, vp, d["prefix_pages"], 20, *meta)
    with torch.no_grad():
        assert torch.equal(q4b.prefix_attention(grad(q), kp, vp, d["prefix_pages"], 20, *meta), ref)


# ---- results over inputs ----------------------------------------------------------------------------------


def test_verify_refuses_results_over_tokens(q4b):  # noqa: F811
    toks, qs = torch.zeros(5, dtype=torch.int32, device=DEV), torch.tensor([0, 3, 5], dtype=torch.int32, device=DEV)
    probs, u = torch.softmax(torch.randn(5, 50, device=DEV), -1), torch.rand(5, device=DEV)
    with pytest.raises(q4b.Q4BError, match="overlap"):
        q4b.verify_drafts(probs, None, toks, u, qs, out=toks)
    both = torch.zeros(10, dtype=torch.int32, device=DEV)  # neighbours in one buffer are apart
    a, _ = q4b.verify_drafts(probs, None, both[:5], u, qs, out=both[5:])
    b, _ = q4b.verify_drafts(probs, None, toks, u, qs)
    assert torch.equal(a, b)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,fused", [(700, False), (1, True)])
def test_append_rotates_q_in_place(q4b, layout, rows, fused):  # noqa: F811
    """q_out = q: contiguous, or the one row of a fused projection."""
    b, q, k, v, kp, vp, cos, sin = _append_case([(rows, rows + 9)], 16, 3, 8, 2, 64, 32, "float16", "float16", 3)
    d = _dev(b)
    meta = (d["page_table"], d["seq_lens"], d["q_start"], cos, sin)
    kw = dict(prefix_len=3, layout=layout)
    ref = q4b.paged_rope_append(q, k, v, kp, vp, *meta, **kw)
    k0, v0 = kp.clone(), vp.clone()
    q2 = q if fused else q.contiguous()
    assert q4b.paged_rope_append(q2, k, v, kp, vp, *meta, q_out=q2, **kw) is q2
    assert torch.equal(q2, ref) and torch.equal(kp, k0) and torch.equal(vp, v0)
    with pytest.raises(q4b.Q4BError, match="overlap"):
        wide = torch.zeros(rows * 8 * 64 + 64, dtype=torch.float16, device=DEV)
        q4b.paged_rope_append(wide[:-64].view(-1, 8, 64), k, v, kp, vp, *meta, q_out=wide[64:].view(-1, 8, 64), **kw)


# ---- prefix_attention: which kernels run ------------------------------------------------------------------


@pytest.fixture(scope="module")
def kernels():
    """The kernels of some calls, by torch's profiler in a process of its own (one profiler session can leave the next one in the
    same process without events)."""
    import json
    import pathlib
    import subprocess
    import sys
    here = pathlib.Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, str(here / "batch_kernels_worker.py")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return json.loads(r.stdout.strip().splitlines()[-1])


def _steps():
    """Steps with many rows: name -> (arguments of _attend_case, keyword arguments of the call)."""
    many = ([(20, 70), (30, 40), (1, 8)], 16, 6000, 16, 8)
    chunk = ([(180, 700), (1, 90)] + [(0, 5)] * 190, 16, 0, 16, 4, 64, torch.float16)
    got = {f"many {hd} {dtype}": ((*many, hd, dtype), {}) for hd in (64, 128) for dtype in (torch.float16, torch.bfloat16)}
    return {**got, "chunk told": (chunk, dict(max_new=180)), "chunk as single tokens": (chunk, dict(max_new=1))}


def _odd(q):
    """q where the tensor-core kernel does not read it: rows that do not begin at 16 bytes."""
    rows, H, hd = q.shape
    return torch.empty(rows, H * hd + 2, dtype=q.dtype, device=DEV)[:, 2:].view(rows, H, hd).copy_(q)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_rows_run_on_the_tensor_core_kernel(q4b, kernels, hd, dtype):  # noqa: F811
    """In this build the tensor-core kernel has the registers of its split, so the plan uses it; and a step that it is not
    used for (here for its q) runs on the other kernels with the same results."""
    name = f"many {hd} {dtype}"
    on, off = kernels[name], kernels[name + " odd"]
    assert any("prefix_tc_kernel" in k for k in on), on
    assert not any("prefix_tc_kernel" in k for k in off) and any("prefix_narrow_kernel" in k for k in off), off
    b, q, kp, vp = _attend_case(*_steps()[name][0], 5)
    _run_attend(q4b, (b, _odd(q), kp, vp), 16)


@pytest.mark.parametrize("lens,prefix,width", [
    ([(180, 700), (1, 90), (1, 1)] + [(0, 5)] * 190, 0, 50),  # fewer rows than sequences, most of them in one
    ([(180, 700), (1, 90), (1, 1)] + [(0, 5)] * 190, 5000, 50),
    ([(1, 200)] * 33, 2500, 400),  # tables much wider than the sequences
    ([(3, 70), (5, 9), (1, 300)] * 8, 3000, 300),
])
def test_told_lengths_change_no_result(q4b, lens, prefix, width):  # noqa: F811
    """max_new and own_keys, right or far off, choose kernels and SMs only."""
    n_pages = sum(-(-o // 16) for _, o in lens) + -(-prefix // 16) + 2
    b = R.make_batch(lens, 16, n_pages, prefix_len=prefix, width=width)
    g = torch.Generator(device=DEV).manual_seed(width)
    q = torch.randn(b["rows"], 16, 64, generator=g, device=DEV).half()
    kp, vp = (torch.randn(n_pages, 16, 4, 64, generator=g, device=DEV).half() for _ in range(2))
    most, mean = max(n for n, _ in lens), int(np.mean([o for _, o in lens]))
    for kw in ({}, dict(max_new=most, own_keys=mean), dict(max_new=1), dict(max_new=2**31 - 1, own_keys=1),
               dict(own_keys=2**31 - 1)):
        d = _dev(b)
        out = _f64(q4b.prefix_attention(q, kp, vp, d["prefix_pages"], prefix, d["page_table"], d["seq_lens"], d["q_start"], **kw))
        ref = R.attention(_f64(q), _f64(kp), _f64(vp), b, 16) if not kw else ref
        _check_attend(out.reshape(ref.shape), ref, _f64(vp), torch.float16, np.ones(b["rows"], dtype=bool))
    for bad in (dict(max_new=-1), dict(own_keys="x")):
        with pytest.raises(ValueError, match=next(iter(bad))):
            q4b.prefix_attention(q, kp, vp, d["prefix_pages"], prefix, d["page_table"], d["seq_lens"], d["q_start"], **bad)


def test_a_told_prompt_chunk_runs_on_the_tensor_cores(kernels):
    assert any("prefix_tc_kernel" in k for k in kernels["chunk told"])
    assert not any("prefix_tc_kernel" in k for k in kernels["chunk as single tokens"])


# ---- malformed offsets, with guards around everything that a call may write -------------------------------


class _Guarded:
    """A tensor inside a larger buffer of a known byte."""

    def __init__(self, shape, dtype, fill=0x5A):
        size = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
        self.raw = torch.full((size + (2 << 20),), fill, dtype=torch.uint8, device=DEV)
        self.size, self.fill = size, fill
        self.t = self.raw[1 << 20:(1 << 20) + size].view(dtype).view(shape)

    def check(self):
        assert bool((self.raw[:1 << 20] == self.fill).all()) and bool((self.raw[(1 << 20) + self.size:] == self.fill).all())


OFFSETS = [[0, 3, 900], [0, 5, 2], [-4, 3, 6], [9, 9, 9], [4, 4, 5], [0, 3, 6]]


def _clamped(offsets, rows):
    """The offsets that the operators go by: clamped to the rows; decreasing ones hold no sequence (attention)."""
    return np.clip(np.array(offsets), 0, rows).astype(np.int32), any(b < a for a, b in zip(offsets, offsets[1:]))


@pytest.mark.parametrize("offsets", OFFSETS)
@pytest.mark.parametrize("rows,prefix,H,Hkv,hd,page", [(6, 50, 8, 2, 64, 8), (6, 50, 4, 2, 32, 20), (6, 30_000, 16, 4, 128, 16),
                                                       (150, 50, 4, 2, 64, 16)])
def test_attend_malformed_offsets_and_guards(q4b, rows, prefix, H, Hkv, hd, page, offsets):  # noqa: F811
    """Rows of no sequence keep what out held, the others follow the clamped offsets, and nothing is written outside out and a
    workspace of exactly the size that was asked for."""
    import ctypes
    from q4b import _lib
    L = _lib.lib()
    own = 44
    b, q, kp, vp = _attend_case([(rows // 2, own), (rows - rows // 2, own)], page, prefix, H, Hkv, hd, torch.float16, 9)
    offsets = [o * rows // 6 for o in offsets]
    d = _dev(b)
    d["q_start"] = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    width = b["page_table"].shape[1]
    # the pool's slots behind the own keys count as keys here: finite ones
    kp, vp = kp.nan_to_num(0.25), vp.nan_to_num(0.5, 0.5, 0.5)
    lens = [2**31 - 1, -5]
    d["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = _Guarded((rows, H * hd), torch.float16)
    out.t.fill_(7.0)
    batch = _lib.Batch(q_start=d["q_start"].data_ptr(), seq_lens=d["seq_lens"].data_ptr(), page_table=d["page_table"].data_ptr(),
                       batch=2, table_width=width, table_stride=width, prefix_len=prefix)
    kv = _lib.PagedKV(k=kp.data_ptr(), v=vp.data_ptr(), dtype=_lib.F16, n_pages=kp.shape[0], page_size=page, n_kv_heads=Hkv,
                      head_dim=hd, page_stride=kp.stride(0), slot_stride=kp.stride(1), head_stride=kp.stride(2))
    need = L.q4b_prefix_attention_workspace(rows, H, ctypes.byref(batch), ctypes.byref(kv))
    ws = _Guarded((need,), torch.uint8)
    rc = L.q4b_prefix_attention(q.data_ptr(), H * hd, hd, rows, H, hd**-0.5, d["prefix_pages"].data_ptr(), ctypes.byref(batch),
                                ctypes.byref(kv), out.t.data_ptr(), ws.t.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, L.q4b_last_error()
    torch.cuda.synchronize()
    out.check(), ws.check()
    q_start, bad = _clamped(offsets, rows)
    if bad:
        assert bool((out.t == 7.0).all())
        return
    far = width * page + rows + 1
    wide = np.concatenate([b["page_table"], np.full((2, -(-far // page) - width), -1, dtype=np.int32)], 1)
    ref = R.attention(_f64(q), _f64(kp), _f64(vp), dict(b, q_start=q_start, page_table=wide,
                                                        seq_lens=np.array([min(x, far) if x > 0 else 0 for x in lens])), page)
    live = ~np.isnan(ref).any(axis=(1, 2))
    got = _f64(out.t).reshape(ref.shape)
    assert (got[~live] == 7.0).all()
    _check_attend(np.where(live[:, None, None], got, 0), np.where(live[:, None, None], ref, 0), _f64(vp), torch.float16, live)


@pytest.mark.parametrize("offsets", OFFSETS)
def test_append_and_verify_malformed_offsets_and_guards(q4b, offsets):  # noqa: F811
    rows, H, Hkv, hd, page = 6, 4, 2, 64, 8
    b, q, k, v, kp, vp, cos, sin = _append_case([(3, 30), (3, 44)], page, 0, H, Hkv, hd, 64, "float16", "float16", 9)
    d = _dev(b)
    q_start, bad = _clamped(offsets, rows)
    qs = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    gk, gv, out = _Guarded(kp.shape, kp.dtype), _Guarded(vp.shape, vp.dtype), _Guarded((rows, H, hd), q.dtype)
    gk.t.copy_(kp), gv.t.copy_(vp), out.t.fill_(7.0)
    q4b.paged_rope_append(q, k, v, gk.t, gv.t, d["page_table"], d["seq_lens"], qs, cos, sin, q_out=out.t)
    for x in (gk, gv, out):
        x.check()
    if not bad:
        k0, v0 = _f64(kp), _f64(vp)
        ref = R.append(_f64(q), _f64(k), _f64(v), k0, v0, dict(b, q_start=q_start), _f64(cos), _f64(sin), "half", page)
        live = ~np.isnan(ref).any(axis=(1, 2))
        assert (_f64(out.t)[~live] == 7.0).all()
        _close_rounded(_f64(out.t)[live], ref[live], torch.float16, 2 * np.abs(_f64(q)).max())
        _close_rounded(_f64(gk.t), k0, torch.float16, 2 * np.abs(_f64(k)).max())
        _close_rounded(_f64(gv.t), v0, torch.float16, 0.0)
    target, draft, tokens, uniforms, _ = _verify_case([3, 3], 257, torch.float32, True, 6)
    new = _Guarded((rows,), torch.int32)
    new.t.fill_(77)
    _, acc = q4b.verify_drafts(target, draft, tokens, uniforms, qs, out=new.t)
    new.check()
    if bad:
        assert all(0 <= a <= rows for a in acc.tolist())
        return
    n = lambda t: t.cpu().numpy()  # noqa: E731
    want, kept = R.verify(n(target), n(draft), n(tokens), n(uniforms), q_start)
    assert acc.tolist() == kept and new.t.tolist() == [77 if w is None else w for w in want]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("factor", [100.0, 230.0, 1000.0])
@pytest.mark.parametrize("lens,prefix,H,Hkv,hd,page", [
    ([(1, 300), (1, 9)], 0, 4, 1, 128, 16), ([(3, 300)], 0, 8, 2, 64, 16), ([(2, 300)], 0, 8, 2, 64, 20), ([(30, 300)], 0, 4, 2, 32, 16),
    ([(1, 1)] * 40, 4000, 8, 2, 128, 16), ([(30, 300)], 0, 16, 2, 64, 16)])
def test_scores_of_many_millions(q4b, lens, prefix, H, Hkv, hd, page, factor, dtype):  # noqa: F811
    """Scores so large that fp32 steps by 1/2 to 4 beside them, in base 2: the key with the largest has all the weight, and the
    result is its V, but for one rounding of the weight and one of the result."""
    n_pages = -(-prefix // page) + sum(-(-o // page) for _, o in lens)
    b = R.make_batch(lens, page, n_pages, prefix_len=prefix)
    g = torch.Generator(device=DEV).manual_seed(1)
    kp = torch.zeros(n_pages, page, Hkv, hd, dtype=dtype, device=DEV)
    vp = torch.randn(n_pages, page, Hkv, hd, generator=g, device=DEV).to(dtype)
    kp[..., 0] = 30464.0
    q = torch.zeros(b["rows"], H, hd, dtype=dtype, device=DEV)
    q[:, :, 0] = factor
    d = _dev(b)
    want = torch.empty(b["rows"], H, hd, dtype=dtype, device=DEV)
    for i, (n, o) in enumerate(lens):
        pages, at = (b["prefix_pages"], prefix // 3) if prefix else (b["page_table"][i], (o - n) // 2)
        kp[pages[at // page], at % page, :, 0] = 40960.0
        want[b["q_start"][i]:b["q_start"][i + 1]] = vp[pages[at // page], at % page].repeat_interleave(H // Hkv, 0)
    got = q4b.prefix_attention(q, kp, vp, d["prefix_pages"], prefix, d["page_table"], d["seq_lens"], d["q_start"], scale=1.0)
    err = (got.view(want.shape).float() - want.float()).abs()
    assert bool((err <= (torch.finfo(dtype).eps + 2.0**-15) * want.float().abs()).all())


# ---- steps one behind the other -----------------------------------------------------------------------------


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("B,new,prefix,H,Hkv,hd", [(32, 1, 2048, 24, 8, 128), (40, 4, 3000, 16, 4, 64), (6, 60, 500, 8, 2, 128), (20, 2, 0, 8, 2, 64)])
def test_steps_in_a_row_see_what_the_last_one_wrote(q4b, B, new, prefix, H, Hkv, hd, graph):  # noqa: F811
    """Decode steps without a pause: projections, lengths and offsets change in the same tensors right in front of each append, and
    the attention of each step (two kernels that overlap, started early) gives the bits of a step that waits for everything."""
    page, steps, rows = 16, 12, B * new
    n_prefix, width = -(-prefix // page), -(-(40 + steps * new) // page)
    g = torch.Generator(device=DEV).manual_seed(B)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).half()  # noqa: E731
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)  # noqa: E731
    rng = np.random.default_rng(B)
    ids = rng.permutation(n_prefix + B * width)
    pages, table = i32(ids[:n_prefix]), i32(ids[n_prefix:].reshape(B, width))
    pools = [rn(len(ids), page, Hkv, hd) for _ in range(2)]
    qkv = [rn(rows, (H + 2 * Hkv) * hd) for _ in range(steps)]
    news = [rng.integers(0, new + 1, B) for _ in range(steps)]  # a step's rows, some sequences idle
    first = rng.integers(1, 40, B)
    starts = [i32(np.concatenate([[0], np.cumsum(n)])) for n in news]
    lens = [i32(first + np.sum(news[:s + 1], 0)) for s in range(steps)]
    now = dict(qkv=torch.empty_like(qkv[0]), start=torch.empty_like(starts[0]), lens=torch.empty_like(lens[0]),
               q=torch.empty(rows, H, hd, dtype=torch.float16, device=DEV))

    def run(kp, vp, s, wait):
        done = torch.cuda.synchronize if wait else lambda: None
        for name, src in (("qkv", qkv), ("start", starts), ("lens", lens)):
            now[name].copy_(src[s])
        done()
        q, k, v = (x.view(rows, -1, hd) for x in now["qkv"].split([H * hd, Hkv * hd, Hkv * hd], 1))
        q4b.paged_rope_append(q, k, v, kp, vp, table, now["lens"], now["start"], prefix_len=prefix, q_out=now["q"])
        done()
        return q4b.prefix_attention(now["q"], kp, vp, pages, prefix, table, now["lens"], now["start"],
                                    out=torch.zeros(rows, H * hd, dtype=torch.float16, device=DEV))

    slow = [x.clone() for x in pools]
    want = [run(*slow, s, True).clone() for s in range(steps)]
    fast = [x.clone() for x in pools]
    torch.cuda.synchronize()
    if graph:
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            got = [run(*fast, s, False) for s in range(steps)]
        for _ in range(3):
            for x, y in zip(fast, pools):
                x.copy_(y)
            cg.replay()
    else:
        got = [run(*fast, s, False) for s in range(steps)]
    torch.cuda.synchronize()
    for s in range(steps):
        assert torch.equal(got[s], want[s]), s
    assert all(torch.equal(x, y) for x, y in zip(fast, slow))


@pytest.mark.parametrize("B,new,prefix,H,Hkv,hd", [(27, 1, 2048, 24, 8, 128), (37, 1, 3000, 24, 8, 64), (9, 40, 0, 8, 2, 128),
                                                   (12, 3, 60, 8, 2, 64), (9, 3, 60, 8, 2, 32)])
def test_padding_rows_change_no_bit_of_others(q4b, B, new, prefix, H, Hkv, hd):  # noqa: F811
    """What q holds in rows of no sequence: zeros, numbers, large ones, NaN, infinities."""
    b, q, kp, vp = _attend_case([(new, 40)] * B, 16, prefix, H, Hkv, hd, torch.float16, 1, spare=30)
    d, n = _dev(b), B * new
    got = []
    for pad in (torch.zeros_like(q[n:]), 3 * torch.randn_like(q[n:]), 200 * torch.randn_like(q[n:]), float("nan"), float("inf")):
        q[n:] = pad
        got.append(q4b.prefix_attention(q, kp, vp, d["prefix_pages"], prefix, d["page_table"], d["seq_lens"], d["q_start"])[:n].clone())
    for x in got[1:]:
        assert torch.equal(x, got[0])


# ---- calls of real length, and orders that are allowed ------------------------------------------------------


def _attend64(q, kp, vp, b, page):
    """The 64-bit form on the GPU, a sequence at a time; every page is there."""
    rows, H, hd = q.shape
    Hkv = kp.shape[2]
    pick = lambda pool, pages, n: pool[torch.from_numpy(np.asarray(pages)).long().to(DEV)].reshape(-1, Hkv, hd)[:n].double()  # noqa: E731
    out = torch.full((rows, H, hd), float("nan"), dtype=torch.float64, device=DEV)
    p = b["prefix_len"]
    for i, n in enumerate(b["seq_lens"].tolist()):
        lo, hi = int(b["q_start"][i]), int(b["q_start"][i + 1])
        own = b["page_table"][i][:-(-n // page)]
        k, v = (torch.cat([pick(x, b["prefix_pages"], p), pick(x, own, n)]) for x in (kp, vp))
        at = torch.arange(p + n, device=DEV)
        for t in range(lo, hi, 64):  # some rows at a time
            r = torch.arange(t, min(t + 64, hi), device=DEV)
            s = torch.einsum("thgd,khd->hgtk", q[r].double().view(len(r), Hkv, H // Hkv, hd), k) / hd**0.5
            s.masked_fill_(at > (p + n - (hi - lo) + r - lo)[:, None], -torch.inf)
            out[r] = torch.einsum("hgtk,khd->thgd", s.softmax(-1), v).reshape(len(r), H, hd)
    return out.cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,prefix,H,Hkv,hd,page", [
    ([(2600, 2600)], 0, 8, 2, 128, 16),  # the fill of a prefix: causal rows only
    ([(1, 100_000), (3, 40_001)], 0, 8, 2, 64, 16),  # long own contexts
    ([(700, 33_000), (1, 20_000)], 1000, 8, 2, 128, 64),
    ([(5, 12_345)] * 3, 0, 8, 8, 32, 20),
])
def test_attend_long(q4b, lens, prefix, H, Hkv, hd, page, dtype):  # noqa: F811
    b, q, kp, vp = _attend_case(lens, page, prefix, H, Hkv, hd, dtype, 17)
    d = _dev(b)
    ref = _attend64(q, kp, vp, b, page)
    got = _f64(q4b.prefix_attention(q, kp, vp, d["prefix_pages"], prefix, d["page_table"], d["seq_lens"], d["q_start"]))
    _check_attend(got.reshape(ref.shape), ref, _f64(vp[:64]), dtype, np.ones(len(ref), dtype=bool))


@pytest.mark.parametrize("lens,prefix,H,Hkv,hd,page", [([(1, 30)] * 70, 4000, 8, 2, 128, 16), ([(90, 300), (2, 40)], 100, 8, 2, 64, 16),
                                                       ([(2, 30)] * 5, 60, 8, 2, 64, 16), ([(20, 30)] * 5, 60, 8, 2, 32, 20)])
def test_attend_orders_of_q_shared_pages_and_out_over_q(q4b, lens, prefix, H, Hkv, hd, page):  # noqa: F811
    """In every kernel: q head-major or one row for all, pages that several places of the tables name, and the result over q."""
    b, q, kp, vp = _attend_case(lens, page, prefix, H, Hkv, hd, torch.float16, 23)
    kp, vp = kp.nan_to_num(0.0), vp.nan_to_num(0.0, 0.0, 0.0)
    b["prefix_pages"][1::2] = b["prefix_pages"][::2][:len(b["prefix_pages"][1::2])]
    b["page_table"][:] = b["page_table"][0]  # every sequence in the first one's pages
    b["page_table"][:, -1] = b["page_table"][0, 0]
    d = _dev(b)
    call = lambda x, **kw: q4b.prefix_attention(x, kp, vp, d["prefix_pages"], prefix, d["page_table"], d["seq_lens"], d["q_start"], **kw)  # noqa: E731
    ref = _attend64(q, kp, vp, b, page)
    want = call(q)
    _check_attend(_f64(want).reshape(ref.shape), ref, _f64(vp), torch.float16, np.ones(len(ref), dtype=bool))
    assert torch.equal(call(q.transpose(0, 1).contiguous().transpose(0, 1)), want)
    assert torch.equal(call(q[:1].expand_as(q)), call(q[:1].expand_as(q).contiguous()))
    q2 = q.clone()
    out = q2.view(len(q2), -1)
    assert call(q2, out=out) is out and torch.equal(out, want)
