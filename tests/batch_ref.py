"""Plain 64-bit implementations of the batched serving operators on the CPU, written from their formulas:
what the GPU tests compare with."""

import math

import numpy as np
import torch


def make_batch(lens, page_size, n_pages, prefix_len=0, width=None, seed=0, spare_rows=0):
    """lens: (new rows, own keys) per sequence -> host arrays of a ragged batch over shuffled pages."""
    rng = np.random.default_rng(seed)
    need = [-(-own // page_size) for _, own in lens]
    n_prefix = -(-prefix_len // page_size)
    ids = rng.permutation(n_pages)[: n_prefix + sum(need)]
    assert len(ids) == n_prefix + sum(need), "not enough pages"
    width = max(need + [1]) if width is None else width
    table = np.full((len(lens), width), -7, dtype=np.int32)  # what nobody may read
    at = n_prefix
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    q_start = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
    return dict(q_start=q_start, seq_lens=np.array([o for _, o in lens], dtype=np.int32), page_table=table,
                prefix_pages=ids[:n_prefix].astype(np.int32), prefix_len=prefix_len, rows=int(q_start[-1]) + spare_rows)


def rotate(x, cos, sin, layout):
    """x [heads, hd] float64, cos / sin [rot / 2] float64."""
    half = cos.shape[0]
    one = np.arange(half) if layout == "half" else 2 * np.arange(half)
    two = one + half if layout == "half" else one + 1
    y = x.copy()
    y[:, one] = x[:, one] * cos - x[:, two] * sin
    y[:, two] = x[:, two] * cos + x[:, one] * sin
    return y


def append(q, k, v, kp, vp, batch, cos, sin, layout, page_size):
    """float64 arrays; kp, vp [n_pages, page_size, Hkv, hd] are written; returns q_out (NaN rows: untouched)."""
    out = np.full(q.shape, np.nan)
    for b in range(len(batch["seq_lens"])):
        lo, hi = batch["q_start"][b], batch["q_start"][b + 1]
        for t in range(lo, hi):
            s = int(batch["seq_lens"][b]) - (hi - lo) + (t - lo)
            pos = batch["prefix_len"] + s
            if cos is not None and not 0 <= pos < len(cos):
                out[t] = 0.0
                continue
            out[t] = q[t] if cos is None else rotate(q[t], cos[pos], sin[pos], layout)
            if 0 <= s < batch["page_table"].shape[1] * page_size:
                page = batch["page_table"][b, s // page_size]
                if 0 <= page < len(kp):
                    kp[page, s % page_size] = k[t] if cos is None else rotate(k[t], cos[pos], sin[pos], layout)
                    vp[page, s % page_size] = v[t]
    return out


def attention(q, kp, vp, batch, page_size, scale=None):
    """float64 q [rows, H, hd], pools; returns [rows, H, hd] (NaN rows: untouched). Masked keys are left out, so
    whatever stands in them cannot matter."""
    rows, H, hd = q.shape
    g = H // kp.shape[2]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    out = np.full(q.shape, np.nan)

    def keys(table, n):
        got = [(table[s // page_size], s % page_size) for s in range(n)]
        got = [(p, o) for p, o in got if 0 <= p < len(kp)]
        at = [i for i, s in enumerate(range(n)) if 0 <= table[s // page_size] < len(kp)]
        p, o = np.array([x for x, _ in got], dtype=np.int64), np.array([x for _, x in got], dtype=np.int64)
        return kp[p, o], vp[p, o], np.array(at, dtype=np.int64)

    pk, pv, _ = keys(batch["prefix_pages"], batch["prefix_len"])
    for b in range(len(batch["seq_lens"])):
        lo, hi = batch["q_start"][b], batch["q_start"][b + 1]
        n = int(batch["seq_lens"][b])
        sk, sv, at = keys(batch["page_table"][b], n)
        for t in range(lo, hi):
            see = at <= n - (hi - lo) + (t - lo)
            k, v = np.concatenate([pk, sk[see]]), np.concatenate([pv, sv[see]])
            for h in range(H):
                s = k[:, h // g] @ q[t, h] * scale
                if len(s) == 0:
                    out[t, h] = 0.0
                    continue
                e = np.exp(s - s.max())
                out[t, h] = (e / e.sum()) @ v[:, h // g]
    return out


def verify(target, draft, tokens, uniforms, q_start):
    """numpy arrays (any float type); returns (out_tokens with None where untouched, accepted)."""
    def clean(x):
        x = x.astype(np.float64)
        return np.where(np.isfinite(x) & (x > 0), x, 0.0)

    rows, vocab = target.shape
    out, accepted = [None] * rows, []
    for b in range(len(q_start) - 1):
        lo, hi = int(q_start[b]), int(q_start[b + 1])
        if lo == hi:
            accepted.append(0)
            continue
        kept = 0
        for r in range(lo, hi - 1):
            x = int(tokens[r + 1])
            if not 0 <= x < vocab:
                break
            d = 1.0 if draft is None else clean(draft[r, x])
            if not float(uniforms[r]) * float(d) < float(clean(target[r, x])):
                break
            kept += 1
        r = lo + kept
        w = clean(target[r])
        if r < hi - 1:
            rest = w.copy()
            if draft is not None:
                rest = np.maximum(w - clean(draft[r]), 0.0)
            elif 0 <= tokens[r + 1] < vocab:
                rest[tokens[r + 1]] = 0.0
            if rest.sum() > 0:
                w = rest
        acc = np.cumsum(w)
        above = np.nonzero(acc > float(uniforms[hi - 1]) * acc[-1])[0]
        for i in range(lo, hi):
            out[i] = int(tokens[i + 1]) if i < r else -1
        some = np.nonzero(w > 0)[0]
        out[r] = -1 if not len(some) else int(above[0]) if len(above) else int(some[-1])
        accepted.append(kept)
    return out, accepted


def tensor(a, device, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return t.to(device=device, dtype=dtype or t.dtype)
