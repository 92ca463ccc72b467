"""Batched serving over a paged cache: torch-tensor wrappers over the C ABI's batch entry points (no
reference counterpart: scripts/llm/llama_q4.py serves one request).

A step of a ragged batch is described by tensors on the device: sequence b has the rows q_start[b] ..
q_start[b + 1] - 1 of the step and, after the step, seq_lens[b] keys of its own, in the pages page_table[b, :],
behind ``prefix_len`` keys that all sequences share. Row j of b is key s = seq_lens[b] - n_b + j at position
prefix_len + s. Rows behind q_start[-1] (a padded step) are left as they were. Every op runs on the
current stream of the tensors' device and can be captured into a CUDA graph, which then follows
what the tensors hold at replay. There is no backward pass: tensors that require grad are refused unless
gradients are off (``torch.no_grad()``)."""

from __future__ import annotations

import ctypes
import importlib

from ._lib import check, lib

_OPS = None


def _ops():
    """The native module, bound to the loaded library (no fallback: a missing build raises)."""
    global _OPS
    if _OPS is None:
        import torch  # noqa: F401  its libraries come first
        L = lib()
        try:
            ops = importlib.import_module("._batch_ops", __package__)
        except ModuleNotFoundError as e:
            raise ImportError("q4b._batch_ops is not built; build it with "
                              "`make -C iree-adreno-genai-tuner_b200/csrc` or __graft_entry__.build()") from e
        ops.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            L.q4b_paged_rope_append, L.q4b_prefix_attention_workspace, L.q4b_prefix_attention, L.q4b_verify_drafts)))
        _OPS = ops
    return _OPS


def paged_rope_append(q, k, v, k_pages, v_pages, page_table, seq_lens, q_start, cos=None, sin=None, *,
                      prefix_len: int = 0, layout: str = "half", q_out=None):
    """Append a step's keys and values to the paged cache, q and k rotated on the way; returns the rotated q.

    q [rows, H, hd], k and v [rows, Hkv, hd] fp32 or of the cache's type (views into one fused
    projection's rows are fine); k_pages, v_pages [n_pages, page_size, Hkv, hd] fp16 or bf16, written in
    place; cos, sin fp32 [positions, rot / 2] (``rope_tables(...)[i][:, : rot // 2]``, or tables of any
    scaling): the first ``rot`` elements of a head turn, as pairs (i, i + rot / 2) with layout "half" and
    (2 i, 2 i + 1) with "interleaved"; None turns nothing. The rotated q is [rows, H, hd] of the cache's type
    (``q_out`` if given; it may be q itself). head_dim and rot are multiples of 16.

    The step's rows come last in their sequences: seq_lens counts them. To fill the shared prefix itself,
    call with prefix_len = 0 and page_table = prefix_pages[None]."""
    r = (_OPS or _ops()).paged_rope_append(q, k, v, k_pages, v_pages, page_table, seq_lens, q_start, cos, sin,
                                           prefix_len, layout, q_out)
    if r.__class__ is int:
        check(r, "paged_rope_append")
    return r


def prefix_attention(q, k_pages, v_pages, prefix_pages, prefix_len: int, page_table, seq_lens, q_start, *,
                     scale=None, out=None, max_new=None, own_keys=None):
    """Attention of a step's rows over the shared prefix and each sequence's own keys -> [rows, H * hd].

    q [rows, H, hd] of the cache's type, rotated (any row and head stride); prefix_pages int32: the pages
    of the prefix_len shared keys (prefix_len 0: none, every sequence on its own). Row j of sequence b sees the
    prefix and b's own keys up to its own; a row that sees none is zero. The prefix is read
    once for all sequences. scale defaults to 1 / sqrt(hd). head_dim 32, 64 or 128.

    max_new and own_keys, where the caller knows them, choose among kernels (results differ by the order of sums alone): the most rows of any
    sequence (else 1 if rows <= B, so a step of one prompt chunk and many idle sequences wants it), and about how many
    own keys a sequence has (else half of what a row of page_table holds, so tables much wider than the sequences want it)."""
    r = (_OPS or _ops()).prefix_attention(q, k_pages, v_pages, prefix_pages, prefix_len, page_table, seq_lens, q_start,
                                          scale, out, max_new, own_keys)
    if r.__class__ is int:
        check(r, "prefix_attention")
    return r


def verify_drafts(target, draft, tokens, uniforms, q_start, *, out=None):
    """Verify drafted tokens against the target's probabilities; returns (tokens [rows], accepted [B]) int32.

    target [rows, V] and draft [rows, V] (or None: drafts without probabilities of their own) fp32, fp16 or
    bf16: row r is the distribution of the token behind row r. tokens int32 [rows]: the step's input tokens,
    the first row of a sequence its last sure token, the others its drafts. uniforms fp32 [rows] in [0, 1):
    row r decides on tokens[r + 1], a sequence's last row draws the new token. Returned at a sequence's
    rows: its kept drafts, the drawn token, then -1; ``accepted`` counts the kept drafts. ``out`` takes the tokens
    if given; it may not be ``tokens`` itself.

    Draft x is kept while u * draft[x] < target[x]; the new token is drawn by inversion from the positive part
    of target - draft at the first rejected draft, or from the last row's target if all were kept."""
    r = (_OPS or _ops()).verify_drafts(target, draft, tokens, uniforms, q_start, out)
    if r.__class__ is int:
        check(r, "verify_drafts")
    return r
