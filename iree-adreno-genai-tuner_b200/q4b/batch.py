"""Batched serving over a paged cache: torch-tensor wrappers over the C ABI's batch entry points (no
reference counterpart: scripts/llm/llama_q4.py serves one request).

A step of a ragged batch is described by tensors on the device: sequence b has the rows q_start[b] ..
q_start[b + 1] - 1 of the step and, after the step, seq_lens[b] keys of its own, in the pages page_table[b, :],
behind ``prefix_len`` keys that all sequences share. Row j of b is key s = seq_lens[b] - n_b + j at position
prefix_len + s. Rows behind q_start[-1] (a padded step) are left as they were. Every op runs on the
current stream of the tensors' device and can be captured into a CUDA graph, which then follows
what the tensors hold at replay."""

from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from ._lib import BF16, F16, F32, Batch, PagedKV, check, lib

_DT = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def _same_device(what, **ts):
    dev = None
    for name, t in ts.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{what}: {name} must be a CUDA tensor (there is no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{what}: {name} is on {t.device}, the others on {dev}")
    return dev


def _on(dev):
    return contextlib.nullcontext() if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _int32(what, name, t, dim):
    if t.dtype != torch.int32 or t.dim() != dim or (t.numel() and t.stride(-1) != 1):
        raise ValueError(f"{what}: {name} must be an int32 tensor of {dim} dimension(s), the last contiguous")


def _batch(what, q_start, seq_lens, page_table, prefix_len):
    _int32(what, "q_start", q_start, 1)
    _int32(what, "seq_lens", seq_lens, 1)
    _int32(what, "page_table", page_table, 2)
    n = seq_lens.shape[0]
    if q_start.shape[0] != n + 1 or page_table.shape[0] != n:
        raise ValueError(f"{what}: {n} seq_lens need q_start [{n + 1}] and page_table [{n}, ...]")
    if not 0 <= prefix_len < 2**31:
        raise ValueError(f"{what}: prefix_len {prefix_len}")
    return Batch(q_start.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(), n, page_table.shape[1],
                 page_table.stride(0) if n > 1 else page_table.shape[1], prefix_len)


def _paged_kv(what, k_pages, v_pages):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError(f"{what}: k_pages and v_pages must be [n_pages, page_size, n_kv_heads, head_dim] of one type")
    if k_pages.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{what}: the cache is fp16 or bf16, not {k_pages.dtype}")
    if k_pages.stride() != v_pages.stride() or k_pages.stride(-1) != 1:
        raise ValueError(f"{what}: k_pages and v_pages need the same strides, head_dim contiguous")
    if max(k_pages.shape[:3]) >= 2**31:
        raise ValueError(f"{what}: cache too large")
    return PagedKV(k_pages.data_ptr(), v_pages.data_ptr(), _DT[k_pages.dtype], *k_pages.shape, *k_pages.stride()[:3])


def _rows(what, name, t, heads, dim):
    """[rows, heads, dim] with the heads of a row contiguous -> the stride between rows."""
    if t.dim() != 3 or t.shape[1:] != (heads, dim):
        raise ValueError(f"{what}: {name} must be [rows, {heads}, {dim}]")
    if t.numel() and (t.stride(2) != 1 or (heads > 1 and t.stride(1) != dim)):
        raise ValueError(f"{what}: the heads of a row of {name} must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else heads * dim


def paged_rope_append(q, k, v, k_pages, v_pages, page_table, seq_lens, q_start, cos=None, sin=None, *,
                      prefix_len: int = 0, layout: str = "half", q_out=None):
    """Append a step's keys and values to the paged cache, q and k rotated on the way; returns the rotated q.

    q [rows, H, hd], k and v [rows, Hkv, hd] fp32 or of the cache's type (views into one fused
    projection's rows are fine); k_pages, v_pages [n_pages, page_size, Hkv, hd] fp16 or bf16, written in
    place; cos, sin fp32 [positions, rot / 2] (``rope_tables(...)[i][:, : rot // 2]``, or tables of any
    scaling): the first ``rot`` elements of a head turn, as pairs (i, i + rot / 2) with layout "half" and
    (2 i, 2 i + 1) with "interleaved"; None turns nothing. The rotated q is [rows, H, hd] of the cache's type
    (``q_out`` if given). head_dim and rot are multiples of 16.

    The step's rows come last in their sequences: seq_lens counts them. To fill the shared prefix itself,
    call with prefix_len = 0 and page_table = prefix_pages[None]."""
    what = "paged_rope_append"
    dev = _same_device(what, q=q, k=k, v=v, k_pages=k_pages, v_pages=v_pages, page_table=page_table,
                       seq_lens=seq_lens, q_start=q_start, cos=cos, sin=sin, q_out=q_out)
    kv = _paged_kv(what, k_pages, v_pages)
    batch = _batch(what, q_start, seq_lens, page_table, prefix_len)
    if layout not in ("half", "interleaved"):
        raise ValueError(f"{what}: layout is 'half' or 'interleaved', not {layout!r}")
    if q.dim() != 3:
        raise ValueError(f"{what}: q must be [rows, heads, head_dim]")
    rows, H, hd = q.shape
    if not (k.shape[0] == v.shape[0] == rows) or not (q.dtype == k.dtype == v.dtype):
        raise ValueError(f"{what}: q, k and v need the same rows and type")
    if q.dtype not in (torch.float32, k_pages.dtype):
        raise ValueError(f"{what}: q, k and v are fp32 or of the cache's type, not {q.dtype}")
    qs = _rows(what, "q", q, H, kv.head_dim)
    ks, vs = _rows(what, "k", k, kv.n_kv_heads, kv.head_dim), _rows(what, "v", v, kv.n_kv_heads, kv.head_dim)
    if (cos is None) != (sin is None):
        raise ValueError(f"{what}: cos and sin come together")
    rot = ts = tr = 0
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 or \
                cos.stride() != sin.stride() or (cos.numel() and cos.stride(1) != 1):
            raise ValueError(f"{what}: cos and sin must be fp32 [positions, rot / 2] with the same strides")
        tr, rot, ts = cos.shape[0], 2 * cos.shape[1], cos.stride(0)
    if q_out is None:
        q_out = torch.empty(rows, H, hd, dtype=k_pages.dtype, device=dev)
    elif q_out.shape != q.shape or q_out.dtype != k_pages.dtype or not q_out.is_contiguous():
        raise ValueError(f"{what}: q_out must be a contiguous {k_pages.dtype} tensor of q's shape")
    if rows == 0:
        return q_out
    with _on(dev):
        check(lib().q4b_paged_rope_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _DT[q.dtype], qs, ks, vs, rows, H,
            cos.data_ptr() if rot else None, sin.data_ptr() if rot else None, ts, tr, rot, layout == "interleaved",
            ctypes.byref(batch), ctypes.byref(kv), q_out.data_ptr(), torch.cuda.current_stream().cuda_stream), what)
    return q_out


def prefix_attention(q, k_pages, v_pages, prefix_pages, prefix_len: int, page_table, seq_lens, q_start, *,
                     scale=None, out=None):
    """Attention of a step's rows over the shared prefix and each sequence's own keys -> [rows, H * hd].

    q [rows, H, hd] of the cache's type, rotated (any row and head stride); prefix_pages int32: the pages
    of the prefix_len shared keys (prefix_len 0: none, every sequence on its own). Row j of sequence b sees the
    prefix and b's own keys up to its own; a row that sees none is zero. The prefix is read
    once for all sequences. scale defaults to 1 / sqrt(hd). head_dim 32, 64 or 128."""
    what = "prefix_attention"
    dev = _same_device(what, q=q, k_pages=k_pages, v_pages=v_pages, prefix_pages=prefix_pages, page_table=page_table,
                       seq_lens=seq_lens, q_start=q_start, out=out)
    kv = _paged_kv(what, k_pages, v_pages)
    batch = _batch(what, q_start, seq_lens, page_table, prefix_len)
    _int32(what, "prefix_pages", prefix_pages, 1)
    if prefix_pages.shape[0] * kv.page_size < prefix_len:
        raise ValueError(f"{what}: {prefix_pages.shape[0]} prefix pages of {kv.page_size} hold no {prefix_len} keys")
    if q.dim() != 3 or q.shape[2] != kv.head_dim or q.dtype != k_pages.dtype or (q.numel() and q.stride(2) != 1):
        raise ValueError(f"{what}: q must be [rows, heads, {kv.head_dim}] of the cache's type, head_dim contiguous")
    rows, H, hd = q.shape
    if out is None:
        out = torch.empty(rows, H * hd, dtype=q.dtype, device=dev)
    elif out.shape != (rows, H * hd) or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"{what}: out must be a contiguous {q.dtype} [{rows}, {H * hd}] tensor")
    if rows == 0:
        return out
    L, bp, kp = lib(), ctypes.byref(batch), ctypes.byref(kv)
    with _on(dev):
        # made anew for each call: the allocator keeps streams and captured graphs apart
        ws = torch.empty(L.q4b_prefix_attention_workspace(rows, H, bp, kp), dtype=torch.uint8, device=dev)
        check(L.q4b_prefix_attention(q.data_ptr(), q.stride(0), q.stride(1), rows, H,
                                     1.0 / math.sqrt(hd) if scale is None else scale, prefix_pages.data_ptr(), bp, kp,
                                     out.data_ptr(), ws.data_ptr(), ws.numel(),
                                     torch.cuda.current_stream().cuda_stream), what)
    return out


def verify_drafts(target, draft, tokens, uniforms, q_start, *, out=None):
    """Verify drafted tokens against the target's probabilities; returns (tokens [rows], accepted [B]) int32.

    target [rows, V] and draft [rows, V] (or None: drafts without probabilities of their own) fp32, fp16 or
    bf16: row r is the distribution of the token behind row r. tokens int32 [rows]: the step's input tokens,
    the first row of a sequence its last sure token, the others its drafts. uniforms fp32 [rows] in [0, 1):
    row r decides on tokens[r + 1], a sequence's last row draws the new token. Returned at a sequence's
    rows: its kept drafts, the drawn token, then -1; ``accepted`` counts the kept drafts.

    Draft x is kept while u * draft[x] < target[x]; the new token is drawn by inversion from the positive part
    of target - draft at the first rejected draft, or from the last row's target if all were kept."""
    what = "verify_drafts"
    dev = _same_device(what, target=target, draft=draft, tokens=tokens, uniforms=uniforms, q_start=q_start, out=out)
    _int32(what, "tokens", tokens, 1)
    _int32(what, "q_start", q_start, 1)
    if target.dim() != 2 or target.dtype not in _DT or (target.numel() and target.stride(1) != 1):
        raise ValueError(f"{what}: target must be fp32, fp16 or bf16 [rows, vocab], the last dimension contiguous")
    rows, vocab = target.shape
    if draft is not None and (draft.shape != target.shape or draft.dtype != target.dtype or
                              (draft.numel() and draft.stride(1) != 1)):
        raise ValueError(f"{what}: draft must be like target")
    if tokens.shape[0] != rows or uniforms.shape != (rows,) or uniforms.dtype != torch.float32 or \
            (rows > 1 and uniforms.stride(0) != 1):
        raise ValueError(f"{what}: {rows} rows need int32 tokens [{rows}] and contiguous fp32 uniforms [{rows}]")
    if q_start.shape[0] < 1:
        raise ValueError(f"{what}: q_start must be [batch + 1]")
    n = q_start.shape[0] - 1
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=dev)
    elif out.shape != (rows,) or out.dtype != torch.int32 or not out.is_contiguous():
        raise ValueError(f"{what}: out must be a contiguous int32 [{rows}] tensor")
    accepted = torch.empty(n, dtype=torch.int32, device=dev)
    with _on(dev):
        check(lib().q4b_verify_drafts(
            target.data_ptr(), None if draft is None else draft.data_ptr(), _DT[target.dtype],
            target.stride(0) if rows > 1 else vocab, 0 if draft is None else draft.stride(0) if rows > 1 else vocab,
            vocab, tokens.data_ptr(), uniforms.data_ptr(), rows, q_start.data_ptr(), n, out.data_ptr(),
            accepted.data_ptr(), torch.cuda.current_stream().cuda_stream), what)
    return out, accepted
