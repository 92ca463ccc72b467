"""GPU parity of the batched serving operators against plain 64-bit implementations (tests/batch_ref.py)."""

import numpy as np
import pytest
import torch

import batch_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def q4b():
    import q4b
    return q4b


def _dev(batch):
    return {k: R.tensor(batch[k], DEV) for k in ("q_start", "seq_lens", "page_table", "prefix_pages")}


def _f64(t):
    return t.detach().cpu().double().numpy()


# ---- paged_rope_append -----------------------------------------------------------------------------------

APPEND = [
    # lens (new, own), page, prefix, H, Hkv, hd, rot, layout, source, cache
    ([(1, 1)], 16, 0, 24, 8, 128, 128, "half", "float16", "float16"),
    ([(1, 600)], 16, 1024, 24, 8, 128, 128, "half", "float32", "float16"),
    ([(3, 7), (0, 5), (1, 33), (6, 6)], 16, 100, 8, 2, 64, 32, "interleaved", "float32", "bfloat16"),
    ([(2, 2), (5, 41)], 1, 3, 4, 4, 32, 16, "half", "bfloat16", "bfloat16"),
    ([(37, 37), (1, 20)], 20, 11, 3, 1, 48, 48, "interleaved", "float16", "float16"),
    ([(9, 300)], 7, 0, 2, 2, 256, 64, "half", "float16", "float16"),
    ([(4, 9)], 8, 5, 8, 2, 64, 0, "half", "float32", "float16"),  # nothing turns
    ([(700, 700), (650, 900)], 64, 77, 4, 1, 64, 64, "half", "bfloat16", "bfloat16"),  # several tokens per CTA
]


def _append_case(lens, page, prefix, H, Hkv, hd, rot, src, cache, seed, spare=0):
    b = R.make_batch(lens, page, n_pages=sum(-(-o // page) for _, o in lens) + -(-prefix // page) + 3,
                     prefix_len=prefix, seed=seed, spare_rows=spare)
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    qkv = rn(b["rows"], (H + 2 * Hkv) * hd).to(getattr(torch, src))
    q, k, v = (x.view(b["rows"], -1, hd) for x in qkv.split([H * hd, Hkv * hd, Hkv * hd], 1))
    n_pages = sum(-(-o // page) for _, o in lens) + -(-prefix // page) + 3
    kp, vp = (rn(n_pages, page, Hkv, hd).to(getattr(torch, cache)) for _ in range(2))
    cos = sin = None
    if rot:
        ang = torch.arange(prefix + max(o for _, o in lens), dtype=torch.float64)[:, None] * \
            500000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
        cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    return b, q, k, v, kp, vp, cos, sin


def _close_rounded(got, ref, dtype, terms):
    """One rounding to dtype (half a step: eps / 2 of the value, or half the smallest subnormal) of an fp32 result
    whose two products and one sum are each off by at most half an fp32 step of |a c| + |b s| <= terms."""
    fi = torch.finfo(dtype)
    tol = fi.eps / 2 * np.abs(ref) * (1 + 2**-20) + 3 * 2.0**-24 * terms + fi.tiny * fi.eps / 2
    bad = np.abs(got - ref) > tol
    assert not bad.any(), (np.abs(got - ref)[bad].max(), int(bad.sum()))


def _run_append(q4b, case, layout, page, cache, **kw):
    b, q, k, v, kp, vp, cos, sin = case
    k0, v0 = _f64(kp), _f64(vp)
    d = _dev(b)
    ck, sk = (None, None) if cos is None else (_f64(cos), _f64(sin))
    ref = R.append(_f64(q), _f64(k), _f64(v), k0, v0, b, ck, sk, layout, page)
    out = q4b.paged_rope_append(q, k, v, kp, vp, d["page_table"], d["seq_lens"], d["q_start"], cos, sin,
                                prefix_len=b["prefix_len"], layout=layout, **kw)
    live = ~np.isnan(ref).any(axis=(1, 2))
    dt = getattr(torch, cache)
    _close_rounded(_f64(out)[live], ref[live], dt, 2 * np.abs(_f64(q)).max())
    _close_rounded(_f64(kp), k0, dt, 2 * np.abs(_f64(k)).max())
    _close_rounded(_f64(vp), v0, dt, 0.0)
    return out, live


@pytest.mark.parametrize("lens,page,prefix,H,Hkv,hd,rot,layout,src,cache", APPEND)
def test_append(q4b, lens, page, prefix, H, Hkv, hd, rot, layout, src, cache):
    _run_append(q4b, _append_case(lens, page, prefix, H, Hkv, hd, rot, src, cache, seed=len(lens)), layout, page, cache)


def test_append_leaves_padding_rows_and_other_slots(q4b):
    """Rows behind the last sequence keep what q_out held; slots of no row keep theirs (checked in _run_append
    against pools that were written only where the formulas say)."""
    case = _append_case([(2, 5), (1, 18)], 16, 9, 8, 2, 64, 64, "float16", "float16", 3, spare=4)
    q_out = torch.full((7, 8, 64), 7.0, dtype=torch.float16, device=DEV)
    out, live = _run_append(q4b, case, "half", 16, "float16", q_out=q_out)
    assert out is q_out and live.tolist() == [True] * 3 + [False] * 4
    assert bool((q_out[3:] == 7.0).all())


def test_append_bad_pages_and_far_positions(q4b):
    """A page id outside the pool drops the append, a position that the tables do not reach gives q_out = 0 and
    no append; neither touches anything else."""
    case = list(_append_case([(4, 4), (3, 40), (2, 6)], 4, 2, 4, 2, 32, 32, "float32", "float16", 5))
    b = case[0]
    b["page_table"][0, 0] = 10_000
    b["page_table"][2, 1] = -1
    case[6], case[7] = case[6][:41], case[7][:41]  # positions 2 + 37 .. 2 + 39: the last one is out
    out, _ = _run_append(q4b, tuple(case), "half", 4, "float16")
    assert bool((out[6] == 0).all()) and not bool((out[5] == 0).all())


def test_append_other_orders(q4b):
    """Pools whose pages hold heads before slots, and k and v interleaved in one allocation, are strides."""
    b, q, k, v, kp, vp, cos, sin = _append_case([(3, 30), (1, 4)], 8, 5, 8, 2, 64, 64, "float16", "float16", 9)
    both = torch.randn(kp.shape[0], 2, 2, 8, 64, device=DEV).half()  # [page, k|v, head, slot, hd]
    kp2, vp2 = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    _run_append(q4b, (b, q, k, v, kp2, vp2, cos, sin), "interleaved", 8, "float16")


def test_append_uses_the_models_tables(q4b):
    """cos and sin as q4b.rope_tables makes them (both halves): the first half of the columns, a strided view."""
    cfg = dict(hidden_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=64, rope_theta=500000.0,
               max_position_embeddings=4096)
    cos, sin = (x.to(DEV)[:, :32] for x in q4b.rope_tables(cfg, 64))
    b, q, k, v, kp, vp, _, _ = _append_case([(3, 30), (1, 4)], 8, 5, 8, 2, 64, 64, "float32", "float16", 9)
    _run_append(q4b, (b, q, k, v, kp, vp, cos, sin), "half", 8, "float16")


# ---- prefix_attention ------------------------------------------------------------------------------------

ATTEND = [
    # lens (new, own), page, prefix, H, Hkv, hd
    ([(1, 1)], 16, 0, 24, 8, 128),
    ([(1, 60), (1, 33)], 16, 250, 24, 8, 128),
    ([(1, 0), (0, 9), (1, 1), (1, 64), (1, 65)], 16, 1, 8, 2, 64),  # no own keys, no rows, tile borders
    ([(3, 2), (4, 4), (2, 130)], 8, 0, 6, 1, 64),  # more rows than keys: rows that see nothing
    ([(1, 500)] * 3 + [(1, 3)], 1, 129, 8, 2, 32),
    ([(5, 77), (1, 300), (7, 7)], 20, 63, 32, 4, 64),
    ([(40, 200), (33, 33), (1, 900)], 64, 1000, 3, 1, 128),  # several row tiles, causal inside
    ([(1, 1)] * 70, 16, 513, 8, 8, 128),  # more than one row tile of the prefix, one head per KV head
    ([(2, 2000)], 16, 3000, 8, 2, 128),
    ([(130, 130), (100, 700)], 16, 300, 4, 4, 32),
    # prefixes of whole 128-key tiles and rests, for steps of more than 32 rows per KV head
    ([(1, 5)] * 33, 16, 128, 2, 2, 64),
    ([(1, 40)] * 50, 8, 1290, 8, 2, 64),
    ([(3, 9), (40, 44)], 32, 127, 8, 2, 128),
    ([(1, 1)] * 43, 64, 4096, 6, 2, 128),  # 129 rows: a second tile of one row
    ([(70, 70), (60, 61)], 128, 640, 8, 4, 128),
    ([(2, 2)] * 129, 256, 1000, 2, 1, 64),
    ([(90, 100), (7, 300)], 512, 2200, 3, 1, 128),
    # sequences with many new rows: causal tiles, ends of the keys inside a tile, several row tiles
    ([(200, 200), (5, 300), (1, 700)], 16, 0, 3, 1, 128),
    ([(300, 1000), (2, 1)], 64, 500, 8, 4, 64),
    ([(40, 9), (7, 130), (0, 50), (30, 30)], 8, 0, 6, 2, 64),  # the first rows of 40 see nothing
    ([(1, 1), (129, 129), (128, 128), (127, 400)], 32, 77, 2, 2, 128),
    ([(6, 100)] * 150, 16, 0, 8, 2, 64),  # more items than CTAs
    ([(5, 70)] * 3 + [(1, 900)] * 20, 16, 0, 16, 1, 128),
    # prefixes long enough for the tensor-core kernel (more than 5000 tiles of 16 rows x 64 keys): single tokens and
    # several rows, ends inside a tile, pages smaller and larger than one
    ([(1, 5)] * 150, 16, 4500, 8, 4, 64),
    ([(3, 9), (80, 90)], 32, 6000, 16, 4, 128),
    ([(1, 1)] * 129, 8, 3000, 16, 8, 64),
    ([(2, 40)] * 100, 256, 3500, 8, 8, 128),
    ([(1, 0)] * 40, 128, 12800, 8, 8, 64),  # no own keys; 40 rows; whole tiles
    # a prefix so long that the kernels take turns, its items on a multiple of them of CTAs
    ([(1, 5), (1, 300), (1, 0)], 128, 126_500, 6, 3, 128),
    # pages that are no power of two
    ([(1, 5)] * 150, 24, 4500, 8, 4, 64),
    ([(70, 200), (1, 90), (9, 9)], 48, 333, 3, 1, 128),
    ([(90, 700), (2, 2)], 192, 4000, 16, 4, 128),
    # many rows from pages that no TMA box fits
    ([(70, 200), (1, 90)], 20, 333, 3, 1, 128),
    ([(40, 100)] * 3, 1, 65, 4, 2, 64),
]


def _attend_case(lens, page, prefix, H, Hkv, hd, dtype, seed, spare=0, sharp=1.0):
    n_pages = sum(-(-o // page) for _, o in lens) + -(-prefix // page) + 2
    b = R.make_batch(lens, page, n_pages, prefix_len=prefix, seed=seed, spare_rows=spare)
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    q = (sharp * rn(b["rows"], H, hd)).to(dtype)
    kp, vp = (rn(n_pages, page, Hkv, hd).to(dtype) for _ in range(2))
    # slots that no sequence holds: what a fresh or reused pool may contain
    held = np.zeros((n_pages, page), dtype=bool)
    for pages, n in [(b["prefix_pages"], prefix)] + [(b["page_table"][i], o) for i, (_, o) in enumerate(lens)]:
        for s in range(n):
            held[pages[s // page], s % page] = True
    free = torch.from_numpy(~held).to(DEV)
    kp[free], vp[free] = float("nan"), float("inf")
    return b, q, kp, vp


def _check_attend(got, ref, vp, dtype, live):
    """Output rounding: half a step of the value. P rounding: each weight is off by at most half a step of itself
    (fp16: or half the smallest subnormal), so the weighted mean by eps / 2 * sum(w |v|) <= eps / 2 * max|v|. fp32
    sums and exponentials of scores |s| < 60: below 2^-15 of max|v|."""
    fi = torch.finfo(dtype)
    vmax = np.nanmax(np.abs(np.where(np.isfinite(vp), vp, np.nan)), initial=1.0)
    tol = fi.eps / 2 * np.abs(ref) + (fi.eps / 2 + 2.0**-15) * vmax + fi.tiny * fi.eps
    err = np.abs(got - ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref)) and not (err[live] > tol[live]).any(), np.nanmax(err[live])
    # the bound above is for the worst case; rounding errors of many keys are independent
    if live.any() and np.abs(ref[live]).max() > 0:
        assert np.linalg.norm(err[live]) <= 2 * fi.eps / 2 * np.linalg.norm(ref[live]) + 2.0**-15


def _run_attend(q4b, case, page, **kw):
    b, q, kp, vp = case
    d = _dev(b)
    ref = R.attention(_f64(q), _f64(kp), _f64(vp), b, page, scale=kw.get("scale"))
    out = q4b.prefix_attention(q, kp, vp, d["prefix_pages"], b["prefix_len"], d["page_table"], d["seq_lens"],
                               d["q_start"], **kw)
    live = ~np.isnan(ref).any(axis=(1, 2))
    got = _f64(out).reshape(ref.shape)
    _check_attend(np.where(live[:, None, None], got, 0), np.where(live[:, None, None], ref, 0), _f64(vp), q.dtype, live)
    return out, ref, live


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,page,prefix,H,Hkv,hd", ATTEND)
def test_attend(q4b, lens, page, prefix, H, Hkv, hd, dtype):
    _, _, live = _run_attend(q4b, _attend_case(lens, page, prefix, H, Hkv, hd, dtype, seed=len(lens) + prefix), page)
    assert live.all()


def test_attend_rows_without_keys_are_zero(q4b):
    out, ref, _ = _run_attend(q4b, _attend_case([(3, 1), (2, 0), (1, 5)], 4, 0, 4, 2, 64, torch.float16, 3), 4)
    assert bool((out[:2] == 0).all()) and bool((out[3:5] == 0).all()) and not bool((out[2] == 0).all())


def test_attend_leaves_padding_rows(q4b):
    case = _attend_case([(2, 5), (1, 18)], 16, 40, 8, 2, 64, torch.bfloat16, 3, spare=3)
    case[1][3:] = float("nan")
    out = torch.full((6, 512), 7.0, dtype=torch.bfloat16, device=DEV)
    got, _, live = _run_attend(q4b, case, 16, out=out)
    assert got is out and live.tolist() == [True] * 3 + [False] * 3 and bool((out[3:] == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
def test_attend_bad_prefix_pages_hold_no_keys(q4b, hd, dtype):
    """The same where the prefix runs in tiles: single pages, a whole tile and the first tile missing."""
    for prefix, H, Hkv in ((1000, 8, 4), (6000, 16, 8)):
        case = _attend_case([(20, 70), (30, 40), (1, 8)], 16, prefix, H, Hkv, hd, dtype, 5)
        for i in list(range(8)) + [13] + list(range(24, 32)) + [40, 62]:
            case[0]["prefix_pages"][i] = -1 if i % 2 else 2**31 - 1
        _run_attend(q4b, case, 16)
        case[0]["prefix_pages"][:] = 10**6
        _run_attend(q4b, case, 16)


def test_attend_growing_scores(q4b):
    """Keys ordered by score, so that the running maximum grows from tile to tile, by little and by much."""
    for step, n, heads in ((0.02, 1024, 2), (2.0, 1024, 2), (0.02, 8192, 8), (2.0, 8192, 8)):
        b, q, kp, vp = _attend_case([(1, 9)] * 80, 16, n, heads, heads, 64, torch.float16, 5)
        q[:] = 0
        q[:, :, 0] = 1.0
        pages = torch.from_numpy(b["prefix_pages"]).long().to(DEV)
        kp[pages, :, :, 0] = (torch.arange(n, device=DEV).view(-1, 16, 1) * step).half()
        _run_attend(q4b, (b, q, kp, vp), 16, scale=0.4)


def test_attend_prefix_tiles_from_other_orders(q4b):
    """Head-major pages for the tiled prefix; and a q that the tiles cannot read in 16-byte pieces."""
    b, q, kp, vp = _attend_case([(1, 30)] * 40, 16, 500, 8, 2, 64, torch.float16, 9)
    both = torch.randn(kp.shape[0], 2, 2, 16, 64, device=DEV).half()
    kp2, vp2 = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    kp2.copy_(kp), vp2.copy_(vp)
    wide = torch.randn(40, 520, device=DEV).half()
    q2 = wide[:, 2:514].view(40, 8, 64)
    q2.copy_(q)
    a, _, _ = _run_attend(q4b, (b, q, kp2, vp2), 16)
    c, _, _ = _run_attend(q4b, (b, q2, kp2, vp2), 16)
    assert float((a - c).abs().max()) < 0.01


def test_attend_bad_pages_hold_no_keys(q4b):
    case = _attend_case([(1, 70), (3, 40), (1, 8)], 8, 100, 8, 2, 64, torch.float16, 5)
    case[0]["page_table"][0, 3], case[0]["page_table"][1, 4], case[0]["prefix_pages"][7] = -1, 10**6, 2**31 - 1
    case[0]["page_table"][2, 0] = -2**31
    _run_attend(q4b, case, 8)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,own,g,page", [(4, 20, 4, 8), (4, 4, 1, 8), (60, 100, 3, 8), (150, 290, 2, 8), (4, 20, 4, 20),
                                            (60, 100, 3, 20)])
def test_attend_later_keys_do_not_leak(q4b, value, dtype, new, own, g, page):
    """A draft whose k or v overflowed spoils its own row and later ones, and no earlier row."""
    for which in (0, 1):
        case = _attend_case([(new, own), (2, 9)], page, 30, 2 * g, 2, 64, dtype, 7)
        b, q, kp, vp = case
        bad = own - new + 2  # key of row 2
        (kp, vp)[which][b["page_table"][0, bad // page], bad % page] = value
        d = _dev(b)
        out = _f64(q4b.prefix_attention(q, kp, vp, d["prefix_pages"], 30, d["page_table"], d["seq_lens"], d["q_start"]))
        clean = [t for t in range(b["rows"]) if t < 2 or t >= new]
        with np.errstate(all="ignore"):
            ref = R.attention(_f64(q), _f64(kp), _f64(vp), b, page).reshape(out.shape)
        live = np.zeros(b["rows"], dtype=bool)
        live[clean] = True
        _check_attend(np.where(live[:, None], out, 0), np.where(live[:, None], ref, 0), _f64(vp), dtype, live)
        if which == 1:
            assert not np.isfinite(out[2:new]).any()


def test_attend_strides_scale_and_orders(q4b):
    """q as a part of wider rows and head-major, pools with heads before slots, another scale."""
    b, q, kp, vp = _attend_case([(3, 30), (1, 44)], 8, 50, 8, 2, 64, torch.float16, 9)
    both = torch.randn(kp.shape[0], 2, 2, 8, 64, device=DEV).half()
    kp2, vp2 = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    kp2.copy_(kp), vp2.copy_(vp)
    wide = torch.randn(4, 9 * 64 + 6, device=DEV).half()
    q2 = wide[:, 2:2 + 512].view(4, 8, 64)
    q2.copy_(q)
    _run_attend(q4b, (b, q2, kp2, vp2), 8, scale=0.05)
    q3 = q.transpose(0, 1).contiguous().transpose(0, 1)
    _run_attend(q4b, (b, q3, kp2, vp2), 8)


def test_attend_sharp_scores(q4b):
    """Scores of some hundreds: the running maximum does the work."""
    _run_attend(q4b, _attend_case([(2, 300), (1, 31)], 16, 700, 8, 2, 64, torch.float16, 9, sharp=3.0), 16, scale=2.0)
    _run_attend(q4b, _attend_case([(20, 300), (10, 31)], 16, 700, 8, 2, 64, torch.float16, 9, sharp=3.0), 16, scale=2.0)


@pytest.mark.parametrize("new", [2, 40])
def test_attend_far_pages(q4b, new):
    """Element offsets behind 2^32 in the pool."""
    n_pages, page, Hkv, hd = 70_000, 64, 8, 128  # 4.6e9 elements, 9 GB each
    kp = torch.empty(n_pages, page, Hkv, hd, dtype=torch.float16, device=DEV)
    vp = torch.empty_like(kp)
    b = R.make_batch([(new, 150)], page, 6, prefix_len=100)
    far = np.array([69_999, 3, 65_537, 40_000, 68_000, 66_000])
    for name in ("page_table", "prefix_pages"):
        b[name] = far[b[name]].astype(np.int32)
    g = torch.Generator(device=DEV).manual_seed(0)
    small_k, small_v = (torch.randn(6, page, Hkv, hd, generator=g, device=DEV).half() for _ in range(2))
    at = torch.from_numpy(far).to(DEV)
    kp[at], vp[at] = small_k, small_v
    q = torch.randn(new, 16, hd, generator=g, device=DEV).half()
    d = _dev(b)
    out = _f64(q4b.prefix_attention(q, kp, vp, d["prefix_pages"], 100, d["page_table"], d["seq_lens"], d["q_start"]))
    back = {int(x): i for i, x in enumerate(far)}
    b2 = dict(b, page_table=np.vectorize(back.get)(b["page_table"]), prefix_pages=np.vectorize(back.get)(b["prefix_pages"]))
    ref = R.attention(_f64(q), _f64(small_k), _f64(small_v), b2, page)
    _check_attend(out.reshape(ref.shape), ref, _f64(small_v), torch.float16, np.ones(new, dtype=bool))
    # and the append reaches them
    x = torch.randn(new, 2 * Hkv, hd, device=DEV).half()
    q4b.paged_rope_append(q, x[:, :Hkv], x[:, Hkv:], kp, vp, d["page_table"], d["seq_lens"], d["q_start"], prefix_len=100)
    for j, s in enumerate(range(150 - new, 150)):
        page_id = int(b["page_table"][0, s // page])
        assert torch.equal(kp[page_id, s % page], x[j, :Hkv]) and torch.equal(vp[page_id, s % page], x[j, Hkv:])
    del kp, vp
    torch.cuda.empty_cache()


def test_attend_malformed_offsets_stay_in_bounds(q4b):
    b, q, kp, vp = _attend_case([(3, 30), (3, 44)], 8, 50, 8, 2, 64, torch.float16, 9)
    d = _dev(b)
    for bad in ([0, 3, 900], [0, 5, 2], [-4, 3, 6], [9, 9, 9]):
        q_start = torch.tensor(bad, dtype=torch.int32, device=DEV)
        lens = torch.tensor([2**31 - 1, -5], dtype=torch.int32, device=DEV)
        q4b.prefix_attention(q, kp, vp, d["prefix_pages"], 50, d["page_table"], lens, q_start)
    torch.cuda.synchronize()


# ---- verify_drafts ---------------------------------------------------------------------------------------


def _verify_case(news, vocab, dtype, drafts, seed, sharp=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = sum(news)
    logits = sharp * torch.randn(rows, vocab, generator=g, device=DEV)
    noisy = logits + 0.8 * torch.randn(rows, vocab, generator=g, device=DEV)
    target, draft = torch.softmax(logits, -1), torch.softmax(noisy, -1)
    drawn = torch.multinomial(draft, 1, generator=g)[:, 0].int() if vocab < 2**24 else None
    tokens = torch.cat([drawn[:1], drawn[:-1]])
    q_start = torch.from_numpy(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)).to(DEV)
    return (target.to(dtype), draft.to(dtype) if drafts else None, tokens,
            torch.rand(rows, generator=g, device=DEV), q_start)


def _run_verify(q4b, case, **kw):
    target, draft, tokens, uniforms, q_start = case
    got, acc = q4b.verify_drafts(target, draft, tokens, uniforms, q_start, **kw)
    n = lambda t: t.detach().float().cpu().numpy()  # noqa: E731
    ref, racc = R.verify(n(target), None if draft is None else n(draft), tokens.cpu().numpy(), n(uniforms),
                         q_start.cpu().numpy())
    assert acc.tolist() == racc
    for r, x in enumerate(ref):
        if x is not None:
            assert int(got[r]) == x, r
    return got, acc, ref


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("news,vocab", [([1], 1), ([5], 7), ([3, 1, 0, 6, 2], 1000), ([5] * 3, 32064), ([40, 33], 501),
                                        ([2, 8, 1], 128256), ([3] * 160, 1025), ([4, 4], 49999)])
def test_verify(q4b, news, vocab, drafts, dtype):
    case = _verify_case(news, vocab, getattr(torch, dtype), drafts, seed=vocab + len(news))
    _run_verify(q4b, case)


def test_verify_keeps_every_share(q4b):
    """Over many sequences all lengths of the kept run occur, and the drawn tokens differ from rejected ones."""
    case = _verify_case([4] * 400, 300, torch.float32, True, 11)
    got, acc, _ = _run_verify(q4b, case)
    assert set(acc.tolist()) == {0, 1, 2, 3}


def test_verify_edges(q4b):
    v = 4096
    u = lambda *x: torch.tensor(x, dtype=torch.float32, device=DEV)  # noqa: E731
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    one = torch.zeros(2, v, device=DEV)
    one[:, 5] = 1.0
    # target == draft: always kept (u < 1); then a draw from a single spike, at u = 0 and at the largest u below 1
    for x in (0.0, float(np.nextafter(np.float32(1), np.float32(0)))):
        got, acc, _ = _run_verify(q4b, (one, one, i(0, 5), u(x, x), i(0, 2)))
        assert got.tolist() == [5, 5] and acc.tolist() == [1]
    # a draft of zero probability in both, with an empty residual: rejected, drawn from the target
    got, acc, _ = _run_verify(q4b, (one, one, i(0, 6), u(0.0, 0.5), i(0, 2)))
    assert got.tolist() == [5, -1] and acc.tolist() == [0]
    # drafts outside the vocabulary are not kept
    for x in (-1, v, 2**31 - 1):
        got, acc, _ = _run_verify(q4b, (one, None, i(0, x), u(0.0, 0.5), i(0, 2)))
        assert got.tolist() == [5, -1]
    # no weight anywhere: the token -1; NaN, infinite and negative probabilities count as zero
    zero = torch.zeros(1, v, device=DEV)
    zero[0, 7], zero[0, 8], zero[0, 9] = float("nan"), float("inf"), -1.0
    got, acc, _ = _run_verify(q4b, (zero, None, i(0), u(0.5), i(0, 1)))
    assert got.tolist() == [-1]
    zero[0, 4000] = 1e-30
    got, acc, _ = _run_verify(q4b, (zero, None, i(0), u(0.5), i(0, 1)))
    assert got.tolist() == [4000]


def test_verify_padding_and_strides(q4b):
    """Rows behind the last sequence keep what out held; rows of a wider buffer, p and d aligned differently."""
    target, draft, tokens, uniforms, q_start = _verify_case([3, 2], 1003, torch.float32, True, 4)
    wide = torch.full((8, 1010), float("nan"), device=DEV)
    tw, dw = wide[:, 1:1004], wide.clone()[:, 2:1005]
    tw[:5], dw[:5] = target, draft
    tok = torch.cat([tokens, tokens[:3]])
    uni = torch.cat([uniforms, uniforms[:3]])
    out = torch.full((8,), 77, dtype=torch.int32, device=DEV)
    got, acc, ref = _run_verify(q4b, (tw, dw, tok, uni, q_start), out=out)
    assert got is out and got[5:].tolist() == [77] * 3 and ref[5:] == [None] * 3


def test_verify_malformed_offsets_stay_in_bounds(q4b):
    """q_start beyond the rows or decreasing is clamped on the device: no row outside is touched."""
    target, draft, tokens, uniforms, _ = _verify_case([3, 3], 257, torch.float32, True, 6)
    for bad in ([0, 3, 900], [0, 5, 2], [-4, 3, 6], [9, 9, 9]):
        q_start = torch.tensor(bad, dtype=torch.int32, device=DEV)
        _, acc = q4b.verify_drafts(target, draft, tokens, uniforms, q_start)
        assert all(0 <= a <= 6 for a in acc.tolist())


# ---- the wrappers' refusals, streams, graphs, and a step of them all ---------------------------------------


def test_wrappers_refuse(q4b):
    case = _append_case([(2, 5), (1, 18)], 16, 9, 8, 2, 64, 64, "float16", "float16", 3)
    b, q, k, v, kp, vp, cos, sin = case
    d = _dev(b)
    meta = (d["page_table"], d["seq_lens"], d["q_start"])
    ap = lambda *a, **kw: q4b.paged_rope_append(*a, **{"prefix_len": 9, **kw})  # noqa: E731
    at = lambda *a, **kw: q4b.prefix_attention(*a, **kw)  # noqa: E731
    q16 = q.contiguous()
    bad = [
        (ValueError, "cache's type", lambda: ap(q.bfloat16(), k.bfloat16(), v.bfloat16(), kp, vp, *meta, cos, sin)),
        (ValueError, "same rows", lambda: ap(q, k[:2], v, kp, vp, *meta, cos, sin)),
        (ValueError, "must be \\[rows", lambda: ap(q, k[:, :1], v, kp, vp, *meta, cos, sin)),
        (ValueError, "contiguous", lambda: ap(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, kp, vp, *meta, cos, sin)),
        (ValueError, "together", lambda: ap(q, k, v, kp, vp, *meta, cos, None)),
        (ValueError, "layout", lambda: ap(q, k, v, kp, vp, *meta, cos, sin, layout="both")),
        (ValueError, "fp32 \\[positions", lambda: ap(q, k, v, kp, vp, *meta, cos.half(), sin.half())),
        (ValueError, "same strides", lambda: ap(q, k, v, kp, vp.transpose(1, 2).contiguous().transpose(1, 2), *meta, cos, sin)),
        (ValueError, "int32", lambda: ap(q, k, v, kp, vp, meta[0].long(), *meta[1:], cos, sin)),
        (ValueError, "seq_lens need", lambda: ap(q, k, v, kp, vp, meta[0], meta[1], meta[2][:-1], cos, sin)),
        (ValueError, "out of range", lambda: ap(q, k, v, kp, vp, *meta, cos, sin, prefix_len=-1)),
        (ValueError, "integer", lambda: ap(q, k, v, kp, vp, *meta, cos, sin, prefix_len="9")),
        (ValueError, "CUDA", lambda: ap(q, k, v, kp, vp, meta[0].cpu(), *meta[1:], cos, sin)),
        (ValueError, "q_out", lambda: ap(q, k, v, kp, vp, *meta, cos, sin, q_out=q16.float())),
        (q4b.Q4BError, "rot_dim", lambda: ap(q, k, v, kp, vp, *meta, cos[:, :4], sin[:, :4])),
        (ValueError, "tensor", lambda: at(None, kp, vp, d["prefix_pages"], 9, *meta)),
        (ValueError, "hold no", lambda: at(q16, kp, vp, d["prefix_pages"], 17, *meta)),
        (ValueError, "cache's type", lambda: at(q16.float(), kp, vp, d["prefix_pages"], 9, *meta)),
        (ValueError, "out must", lambda: at(q16, kp, vp, d["prefix_pages"], 9, *meta, out=q16)),
        (q4b.Q4BError, "scale", lambda: at(q16, kp, vp, d["prefix_pages"], 9, *meta, scale=0.0)),
        (TypeError, "number", lambda: at(q16, kp, vp, d["prefix_pages"], 9, *meta, scale="x")),
        (q4b.Q4BError, "head_dim", lambda: at(q16[..., :48], kp[..., :48], vp[..., :48], d["prefix_pages"], 9, *meta)),
        (q4b.Q4BError, "n_kv_heads", lambda: at(q16[:, :3], kp, vp, d["prefix_pages"], 9, *meta)),
    ]
    t, dr, tok, u, qs = _verify_case([3, 2], 100, torch.float32, True, 1)
    bad += [
        (ValueError, "like target", lambda: q4b.verify_drafts(t, dr.half(), tok, u, qs)),
        (ValueError, "like target", lambda: q4b.verify_drafts(t, dr[:, :50], tok, u, qs)),
        (ValueError, "rows need", lambda: q4b.verify_drafts(t, dr, tok[:4], u, qs)),
        (ValueError, "rows need", lambda: q4b.verify_drafts(t, dr, tok, u.double(), qs)),
        (ValueError, "int32", lambda: q4b.verify_drafts(t, dr, tok.long(), u, qs)),
        (ValueError, "last dimension", lambda: q4b.verify_drafts(t.t().contiguous().t(), dr, tok, u, qs)),
        (ValueError, "out", lambda: q4b.verify_drafts(t, dr, tok, u, qs, out=tok[:3])),
    ]
    for kind, word, call in bad:
        with pytest.raises(kind, match=word):
            call()


def test_empty_steps(q4b):
    b, q, k, v, kp, vp, cos, sin = _append_case([(2, 5)], 16, 9, 8, 2, 64, 64, "float16", "float16", 3)
    d = _dev(b)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert q4b.paged_rope_append(q[:0], k[:0], v[:0], kp, vp, d["page_table"], d["seq_lens"], d["q_start"], cos,
                                 sin).shape == (0, 8, 64)
    assert q4b.prefix_attention(q[:0], kp, vp, d["prefix_pages"], 9, d["page_table"][:0], d["seq_lens"][:0], none).shape == (0, 512)
    t, acc = q4b.verify_drafts(torch.zeros(0, 9, device=DEV), None, none[:0], torch.zeros(0, device=DEV), none)
    assert t.numel() == 0 and acc.numel() == 0
    zeros = torch.zeros(4, dtype=torch.int32, device=DEV)  # sequences without rows
    t, acc = q4b.verify_drafts(torch.zeros(0, 9, device=DEV), None, none[:0], torch.zeros(0, device=DEV), zeros)
    assert acc.tolist() == [0, 0, 0]


def _target(s, o):
    """A stand-in for the rest of the model. Not a matrix product of torch's: two graphs captured on one stream share the
    library's workspace, and replayed at once they spoil each other's products."""
    return torch.softmax((o.float()[:, :, None] * s["head"]).sum(1), -1)


def _step(q4b, s):
    """append -> attention -> (a stand-in for the rest of the model) -> verification."""
    q = q4b.paged_rope_append(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lens"], s["q_start"], s["cos"],
                              s["sin"], prefix_len=s["prefix"])
    o = q4b.prefix_attention(q, s["kp"], s["vp"], s["pages"], s["prefix"], s["table"], s["lens"], s["q_start"])
    target = _target(s, o)
    return (q, o) + q4b.verify_drafts(target, s["draft"], s["tokens"], s["uniforms"], s["q_start"])


def _step_case(seed, vocab=500):
    b, q, k, v, kp, vp, cos, sin = _append_case([(3, 30), (1, 44), (5, 5), (2, 100)], 8, 50, 8, 2, 64, 64, "float32",
                                                "float16", seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 100)
    d = _dev(b)
    draft = torch.softmax(torch.randn(11, vocab, generator=g, device=DEV), -1)
    return dict(b=b, q=q, k=k, v=v, kp=kp, vp=vp, cos=cos, sin=sin, table=d["page_table"], lens=d["seq_lens"],
                q_start=d["q_start"], pages=d["prefix_pages"], prefix=50, draft=draft,
                head=0.3 * torch.randn(512, vocab, generator=g, device=DEV),
                tokens=torch.randint(0, vocab, (11,), generator=g, device=DEV, dtype=torch.int32),
                uniforms=torch.rand(11, generator=g, device=DEV))


def test_step_of_a_batch(q4b):
    """The operators in a row, as a serving step runs them, against the plain forms on the way."""
    s = _step_case(21)
    k0, v0 = _f64(s["kp"]), _f64(s["vp"])
    ref_q = R.append(_f64(s["q"]), _f64(s["k"]), _f64(s["v"]), k0, v0, s["b"], _f64(s["cos"]), _f64(s["sin"]), "half", 8)
    q, o, toks, acc = _step(q4b, s)
    _close_rounded(_f64(q), ref_q, torch.float16, 2 * np.abs(_f64(s["q"])).max())
    ref = R.attention(_f64(q), _f64(s["kp"]), _f64(s["vp"]), s["b"], 8)
    _check_attend(_f64(o).reshape(ref.shape), ref, _f64(s["vp"]), torch.float16, np.ones(11, dtype=bool))
    target = _target(s, o).cpu().numpy()
    rt, ra = R.verify(target, s["draft"].cpu().numpy(), s["tokens"].cpu().numpy(), s["uniforms"].cpu().numpy(),
                      s["b"]["q_start"])
    assert toks.tolist() == rt and acc.tolist() == ra


def test_step_in_graphs_and_streams(q4b):
    """Two captured steps replayed on two streams at once, with new contents in the same tensors, give what eager
    calls give; a graph follows lengths and offsets that change between replays."""
    cases = [_step_case(31), _step_case(32)]
    graphs, outs = [], []
    for s in cases:
        _step(q4b, s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(q4b, s))
        graphs.append(g)
    for s, n in zip(cases, (33, 34)):
        new = _step_case(n)
        for name in ("q", "k", "v", "kp", "vp", "draft", "tokens", "uniforms", "head"):
            s[name].copy_(new[name])
        s["lens"].copy_(torch.tensor([17, 40, 5, 93], dtype=torch.int32))
        s["q_start"].copy_(torch.tensor([0, 1, 4, 6, 9], dtype=torch.int32))
    eager = []
    for s in cases:
        kp, vp = s["kp"].clone(), s["vp"].clone()
        eager.append([x.clone() for x in _step(q4b, s)] + [s["kp"].clone(), s["vp"].clone()])
        s["kp"].copy_(kp), s["vp"].copy_(vp)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, out, ref in zip(cases, outs, eager):
        for x, y in zip(list(out) + [s["kp"], s["vp"]], ref):
            live = slice(0, 9) if x.shape[0] == 11 else slice(None)
            assert torch.equal(x[live], y[live])


def test_attend_many_sequences_and_no_tables(q4b):
    """The largest batch that the kernels take, and sequences without pages of their own."""
    _run_attend(q4b, _attend_case([(1, 2), (0, 3), (1, 0), (2, 9)] * 1024, 8, 60, 2, 1, 64, torch.float16, 13), 8)
    b, q, kp, vp = _attend_case([(1, 0), (2, 0)], 16, 40, 4, 2, 64, torch.float16, 3)
    b["page_table"] = b["page_table"][:, :0]
    _run_attend(q4b, (b, q, kp, vp), 16)


def test_large_steps_on_two_streams(q4b):
    """Steps that use the tensor cores, eager and replayed from graphs at once on two streams, with lengths that change."""
    cases = [_attend_case([(1, 100)] * 60 + [(40, 300)], 16, 5000, 16, 4, 128, torch.float16, s) for s in (1, 2)]
    devs = [_dev(c[0]) for c in cases]
    call = lambda c, d: q4b.prefix_attention(c[1], c[2], c[3], d["prefix_pages"], 5000, d["page_table"], d["seq_lens"],  # noqa: E731
                                             d["q_start"])
    graphs, outs = [], []
    for c, d in zip(cases, devs):
        call(c, d)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c, d))
        graphs.append(g)
    for d in devs:
        d["seq_lens"].sub_(torch.arange(61, dtype=torch.int32, device=DEV))
        d["q_start"].copy_(torch.cat([torch.arange(31, dtype=torch.int32), torch.full((30,), 30, dtype=torch.int32),
                                      torch.tensor([70], dtype=torch.int32)]))
    refs = []
    for c, d in zip(cases, devs):
        b = dict(c[0], seq_lens=d["seq_lens"].cpu().numpy(), q_start=d["q_start"].cpu().numpy())
        refs.append(R.attention(_f64(c[1]), _f64(c[2]), _f64(c[3]), b, 16))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    eager = [[], []]
    for n in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                if n % 2:
                    eager[i].append(call(cases[i], devs[i]))
                else:
                    graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        live = ~np.isnan(refs[i]).any(axis=(1, 2))
        assert live[:70].all() and not live[70:].any()
        for o in eager[i] + [outs[i]]:
            got = _f64(o).reshape(refs[i].shape)
            _check_attend(np.where(live[:, None, None], got, 0), np.where(live[:, None, None], refs[i], 0), _f64(cases[i][3]),
                          torch.float16, live)
    assert q4b.lib().q4b_device_status(1) == 0


def test_results_do_not_depend_on_timing(q4b):
    """The same call gives the same bits, whatever runs beside it."""
    s = _step_case(41)
    first = _step(q4b, s)
    side = torch.cuda.Stream()
    noise = torch.randn(4096, 4096, device=DEV)
    for _ in range(10):
        with torch.cuda.stream(side):
            noise @ noise
        for x, y in zip(first, _step(q4b, s)):
            assert torch.equal(x, y)
    torch.cuda.synchronize()
