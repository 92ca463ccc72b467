"""The batched serving operators as measured cases: keys and values appended to a paged cache with the
rotation on the way (``append``), attention of a batch whose sequences share a prefix (``attend``) and the
verification of drafted tokens (``verify``).

A batch is ragged: sequence b has the rows q_start[b] .. q_start[b+1] of a step, and after the step
seq_lens[b] keys of its own, in the pages page_table[b, :], behind prefix_len keys that all sequences share.
"""

import pathlib
import random
import sys

import numpy as np
import torch

own = False

THETA = 500000.0
#: Share of drafted tokens that the target keeps, about; it decides how often a draft row is read.
KEPT = 0.7

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _q4b():
    pkg = str(pathlib.Path(__file__).resolve().parents[1] / "iree-adreno-genai-tuner_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import q4b
    return q4b


# ---- cases -------------------------------------------------------------------------------------


def listed():
    return [
        # one request, one new token: the latency of a step's smallest call
        dict(name="append_one_token", op="append", batch=1, new=1, own_max=600, prefix=1024, heads=24, kv_heads=8,
             dim=128, rot=128, layout="half", page=16, src="fp16", cache="fp16"),
        # drafted tokens of a mid-sized batch: rotation of half of the head, interleaved pairs, fp32 projections
        dict(name="append_drafts", op="append", batch=93, new=6, own_max=900, prefix=2500, heads=32, kv_heads=4,
             dim=64, rot=32, layout="interleaved", page=16, src="fp32", cache="fp16"),
        # chunks of long prompts
        dict(name="append_prompts", op="append", batch=16, new=1100, own_max=1100, prefix=4096, heads=32, kv_heads=8,
             dim=128, rot=128, layout="half", page=64, src="bf16", cache="bf16"),
        # two short chats: latency again
        dict(name="attend_two", op="attend", batch=2, new=1, own_max=60, prefix=250, heads=24, kv_heads=8, dim=128,
             page=16, cache="fp16"),
        # a small decode batch behind a system prompt
        dict(name="attend_decode", op="attend", batch=32, new=1, own_max=512, prefix=2048, heads=24, kv_heads=8,
             dim=128, page=16, cache="fp16"),
        # drafted tokens: several ragged rows for each sequence, odd lengths, small heads
        dict(name="attend_drafts", op="attend", batch=61, new=5, own_max=777, prefix=4099, heads=32, kv_heads=4,
             dim=64, page=16, cache="bf16"),
        # a full decode batch behind a long document
        dict(name="attend_batch", op="attend", batch=192, new=1, own_max=1500, prefix=16384, heads=32, kv_heads=8,
             dim=128, page=16, cache="bf16"),
        # new turns of several chats at once: many rows for each sequence over the shared document
        dict(name="attend_prompts", op="attend", batch=8, new=250, own_max=700, prefix=12001, heads=24, kv_heads=8,
             dim=128, page=64, cache="fp16"),
        # one request with four drafts
        dict(name="verify_one", op="verify", batch=1, new=5, vocab=32064, probs="fp32", drafts=True),
        # a decode batch
        dict(name="verify_batch", op="verify", batch=64, new=6, vocab=128256, probs="fp32", drafts=True),
        # drafts that were looked up in the prompt have no probabilities of their own; an odd vocabulary
        dict(name="verify_lookup", op="verify", batch=155, new=4, vocab=49999, probs="fp16", drafts=False),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "verify"])
    if op == "verify":
        case = dict(op=op, batch=_log(rng, 1, 200), new=rng.randint(1, 8), vocab=_log(rng, 500, 128256),
                    probs=rng.choice(["fp32", "fp32", "fp16", "bf16"]), drafts=rng.random() < 0.7)
        case["batch"] = max(1, min(case["batch"], 64 * 6 * 128256 // (case["vocab"] * case["new"])))
        return case
    heads, kv_heads, dim = rng.choice([(24, 8, 128), (32, 8, 128), (32, 4, 64), (8, 2, 64), (8, 8, 128), (6, 1, 64),
                                       (8, 2, 32)])
    new = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 16, 250)])
    batch = _log(rng, 1, 192)
    if new > 8:
        batch = max(1, min(batch, 2000 // new))
    case = dict(op=op, batch=batch, new=new, own_max=max(_log(rng, 1, 1500), new), prefix=rng.choice([0, _log(rng, 1, 16384),
                _log(rng, 1, 16384)]), heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([1, 8, 16, 16, 20, 32, 64]),
                cache=rng.choice(["fp16", "bf16"]))
    if op == "append":
        case["src"] = rng.choice(["fp32", case["cache"]])
        case["rot"] = rng.choice([dim, dim, dim // 2, 16])
        case["layout"] = rng.choice(["half", "interleaved"])
    return case


def _lengths(case):
    """(new rows, own keys) of each sequence: by the case alone, so that the work is known."""
    r = random.Random(case["batch"] * 7919 + case["new"] * 31 + case.get("own_max", 0))
    got = []
    for b in range(case["batch"]):
        new = case["new"] if case["new"] == 1 or b == 0 else r.randint((case["new"] + 2) // 3, case["new"])
        top = case.get("own_max", new)
        got.append((new, top if b == 0 else r.randint(max(new, top // 4), max(new, top))))
    return got


def work(case):
    lens = _lengths(case)
    rows = sum(n for n, _ in lens)
    if case["op"] == "verify":
        size, v = {"fp32": 4, "fp16": 2, "bf16": 2}[case["probs"]], case["vocab"]
        read = sum(1 + (1 - KEPT ** (n - 1) if case["drafts"] else 0) for n, _ in lens) * v
        return {"bytes": read * size + rows * 20, "flops": 2 * read}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        src = 4 if case["src"] == "fp32" else 2
        return {"bytes": rows * ((h + 2 * hk) * d * (src + 2) + case["rot"] * 4), "flops": rows * (h + hk) * case["rot"] * 3}
    seen = sum(n * (case["prefix"] + own_len - n) + n * (n + 1) // 2 for n, own_len in lens)
    keys = case["prefix"] + sum(own_len for _, own_len in lens)
    return {"bytes": keys * 2 * hk * d * 2 + rows * h * d * 4, "flops": 4 * d * h * seen}


# ---- inputs ------------------------------------------------------------------------------------


def _batch(case, gen, dev):
    """The ragged batch and its pages, in a shuffled pool with some pages that nobody uses."""
    lens = _lengths(case)
    order = torch.randperm(len(lens), generator=gen).tolist()
    lens = [lens[i] for i in order]
    ps, n_prefix = case["page"], -(-case["prefix"] // case["page"])
    new, own_len = np.array([n for n, _ in lens]), np.array([o for _, o in lens])
    pages = -(-own_len // ps)
    width = int(pages.max())
    n_pages = n_prefix + int(pages.sum()) + 7
    ids = torch.randperm(n_pages, generator=gen).numpy()
    table = np.zeros((len(lens), width), dtype=np.int32)
    at = np.arange(width)[None] < pages[:, None]
    table[at] = ids[n_prefix:n_prefix + int(pages.sum())]
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)  # noqa: E731
    return dict(case=case, n_pages=n_pages, rows=int(new.sum()), max_new=int(new.max()), prefix_len=case["prefix"],
                prefix_pages=i32(ids[:n_prefix]), page_table=i32(table), seq_lens=i32(own_len),
                q_start=i32(np.concatenate([[0], np.cumsum(new)])))


def prepare(case, seed):
    dev = torch.device("cuda")
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    if case["op"] == "verify":
        dt, v = _TYPES[case["probs"]], case["vocab"]
        new = np.array([n for n, _ in _lengths(case)])[torch.randperm(case["batch"], generator=host).numpy()]
        q_start = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(dev)
        rows = int(new.sum())
        logits = 3.0 * randn(rows, v)
        drafted = logits + 1.2 * randn(rows, v)
        target = torch.softmax(logits, -1).to(dt)
        # each draft is drawn from the draft model's distribution (largest of logits + Gumbel noise)
        noise = -torch.log(-torch.log(torch.rand(rows, v, generator=gen, device=dev).clamp_(1e-7, 1 - 1e-7)))
        drawn = (drafted + noise).argmax(-1).to(torch.int32)
        tokens = torch.cat([torch.randint(0, v, (1,), generator=gen, device=dev, dtype=torch.int32), drawn[:-1]])
        return dict(case=case, q_start=q_start, tokens=tokens, target=target,
                    draft=torch.softmax(drafted, -1).to(dt) if case["drafts"] else None,
                    uniforms=torch.rand(rows, generator=gen, device=dev))
    s = _batch(case, host, dev)
    h, hk, d, dt = case["heads"], case["kv_heads"], case["dim"], _TYPES[case["cache"]]
    s["k_pages"] = randn(s["n_pages"], case["page"], hk, d).to(dt)
    s["v_pages"] = randn(s["n_pages"], case["page"], hk, d).to(dt)
    if case["op"] == "attend":
        s["q"] = (1.5 * randn(s["rows"], h, d)).to(dt)
        return s
    # q | k | v rows of one fused projection, and the tables of a context scaled to four times its length
    qkv = randn(s["rows"], (h + 2 * hk) * d).to(_TYPES[case["src"]])
    s["q"] = qkv[:, :h * d].view(-1, h, d)
    s["k"] = qkv[:, h * d:(h + hk) * d].view(-1, hk, d)
    s["v"] = qkv[:, (h + hk) * d:].view(-1, hk, d)
    half = case["rot"] // 2
    inv = THETA ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
    ang = torch.arange(case["prefix"] + case["own_max"], dtype=torch.float64, device=dev)[:, None] * (inv / 4)
    s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    return s


# ---- one pass ----------------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        q4b = _q4b()
        if op == "append":
            q_out = q4b.paged_rope_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"],
                                          s["seq_lens"], s["q_start"], s["cos"], s["sin"], prefix_len=s["prefix_len"],
                                          layout=s["case"]["layout"])
            return q_out, s["k_pages"], s["v_pages"]
        if op == "attend":
            return q4b.prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["prefix_pages"], s["prefix_len"],
                                        s["page_table"], s["seq_lens"], s["q_start"])
        return q4b.verify_drafts(s["target"], s["draft"], s["tokens"], s["uniforms"], s["q_start"])
    return {"append": _append, "attend": _attend, "verify": _verify}[op](s)


def _sequence(q_start, rows):
    """For each row: its sequence, and its place in it."""
    row = torch.arange(rows, device=q_start.device, dtype=torch.int32)
    b = torch.searchsorted(q_start, row, right=True) - 1
    return b, row - q_start[b]


def _rotate(x, cos, sin, layout):
    half = cos.shape[-1]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    c, s = cos[:, None, :], sin[:, None, :]
    if layout == "half":
        a, b = rot[..., :half], rot[..., half:]
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    a, b = rot[..., 0::2], rot[..., 1::2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), rest], -1)


def _append(s):
    kp, vp, ps = s["k_pages"], s["v_pages"], s["case"]["page"]
    b, j = _sequence(s["q_start"], s["rows"])
    new = s["q_start"][1:] - s["q_start"][:-1]
    at = s["seq_lens"][b] - new[b] + j
    cos, sin = s["cos"][s["prefix_len"] + at], s["sin"][s["prefix_len"] + at]
    page, slot = s["page_table"][b, at // ps], at % ps
    kp[page, slot] = _rotate(s["k"].float(), cos, sin, s["case"]["layout"]).to(kp.dtype)
    vp[page, slot] = s["v"].to(vp.dtype)
    return _rotate(s["q"].float(), cos, sin, s["case"]["layout"]).to(kp.dtype), kp, vp


def _attend(s):
    kp, vp, p = s["k_pages"], s["v_pages"], s["prefix_len"]
    h, hk, d = s["case"]["heads"], s["case"]["kv_heads"], s["case"]["dim"]
    g, rows, batch, top = h // hk, s["rows"], s["page_table"].shape[0], s["max_new"]
    b, j = _sequence(s["q_start"], rows)
    q = s["q"].float() * d ** -0.5
    # scores against the shared keys: [hk, rows * g, P]
    pk, pv = (x[s["prefix_pages"]].flatten(0, 1)[:p].float().transpose(0, 1) for x in (kp, vp))
    shared = torch.matmul(q.view(rows, hk, g, d).permute(1, 0, 2, 3).reshape(hk, rows * g, d), pk.transpose(1, 2))
    # scores against the own keys, rows padded to the longest sequence: [batch, hk, top * g, keys]
    ok, ov = (x[s["page_table"]].flatten(1, 2).float().transpose(1, 2) for x in (kp, vp))
    keys = ok.shape[2]
    padded = q.new_zeros(batch, top, h, d)
    padded[b, j] = q
    mine = torch.matmul(padded.view(batch, top, hk, g, d).permute(0, 2, 1, 3, 4).reshape(batch, hk, top * g, d),
                        ok.transpose(2, 3)).view(batch, hk, top, g, keys)
    new = (s["q_start"][1:] - s["q_start"][:-1])[:, None]
    last = s["seq_lens"][:, None] - new + torch.arange(top, device=q.device)
    seen = torch.arange(keys, device=q.device) <= last[:, :, None]
    mine = mine.masked_fill(~seen[:, None, :, None, :], float("-inf"))
    mine = mine.permute(0, 2, 1, 3, 4)[b, j].transpose(0, 1).reshape(hk, rows * g, keys)
    both = torch.cat([shared, mine], -1)
    e = torch.exp(both - both.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    out = torch.matmul(w[..., :p], pv).view(hk, rows, g, d).transpose(0, 1)
    own_w = w.new_zeros(batch, top, hk, g, keys)
    own_w[b, j] = w[..., p:].view(hk, rows, g, keys).transpose(0, 1)
    tail = torch.matmul(own_w.permute(0, 2, 1, 3, 4).reshape(batch, hk, top * g, keys), ov)
    out = out + tail.view(batch, hk, top, g, d).permute(0, 2, 1, 3, 4)[b, j]
    return out.reshape(rows, h * d).to(kp.dtype)


def _verify(s):
    p, d, u, start = s["target"], s["draft"], s["uniforms"], s["q_start"]
    rows, batch, v = p.shape[0], start.shape[0] - 1, p.shape[1]
    b, j = _sequence(start, rows)
    new = start[1:] - start[:-1]
    tested = j < new[b] - 1
    x = torch.cat([s["tokens"][1:], s["tokens"][:1]]).long()[:, None]
    px = p.gather(1, x)[:, 0].double()
    dx = d.gather(1, x)[:, 0].double() if d is not None else torch.ones_like(px)
    stop = torch.where(tested & (u.double() * dx < px), v, j)  # a row that ends the accepted run says its own place
    kept = torch.full((batch,), v, dtype=stop.dtype, device=p.device).scatter_reduce(0, b, stop, "amin")
    at = start[:-1] + kept
    w = p[at].double().clamp(min=0)
    cut = (kept < new - 1)[:, None]
    if d is not None:
        rest = (w - d[at].double()).clamp(min=0)
    else:
        rest = w.scatter(1, x[at], 0.0)
    w = torch.where(cut & (rest.sum(-1, keepdim=True) > 0), rest, w)
    acc = w.cumsum(-1)
    pick = (acc <= u[start[1:] - 1].double()[:, None] * acc[:, -1:]).sum(-1)
    some = torch.arange(v, device=p.device).masked_fill(w <= 0, -1).amax(-1)
    pick = torch.minimum(pick, some)
    nxt = torch.cat([s["tokens"][1:], s["tokens"][:1]])
    out = torch.where(j < kept[b], nxt, torch.where(j == kept[b], pick[b].to(torch.int32), -1))
    return out.to(torch.int32), kept.to(torch.int32)


# ---- the definition in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    """Sequence by sequence, from the definitions; the verification has whole numbers alone."""
    if case["op"] == "verify":
        return None
    s = prepare(case, seed)
    ps, p = case["page"], case["prefix"]
    start, lens, table = s["q_start"].tolist(), s["seq_lens"].tolist(), s["page_table"].long()
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "append":
        half = case["rot"] // 2
        if case["layout"] == "half":
            one, two = list(range(half)), list(range(half, 2 * half))
        else:
            one, two = list(range(0, 2 * half, 2)), list(range(1, 2 * half, 2))
        q_out = s["q"].double()
        new_k, kp, vp = s["k"].double(), s["k_pages"].double(), s["v_pages"].double()
        for b in range(len(lens)):
            lo, hi = start[b], start[b + 1]
            own_keys = torch.arange(lens[b] - (hi - lo), lens[b], device=q_out.device)
            cos, sin = (s[n].double()[p + own_keys].unsqueeze(1) for n in ("cos", "sin"))
            for x in (q_out, new_k):
                first, second = x[lo:hi, :, one], x[lo:hi, :, two]
                x[lo:hi, :, one], x[lo:hi, :, two] = first * cos - second * sin, first * sin + second * cos
            where = (table[b, own_keys // ps], own_keys % ps)
            kp[where], vp[where] = new_k[lo:hi], s["v"][lo:hi].double()
        return q_out, kp, vp
    gather = lambda pool, ids, n: pool[ids.long()].reshape(-1, hk, d)[:n]  # noqa: E731
    pk, pv = (gather(s[n], s["prefix_pages"], p) for n in ("k_pages", "v_pages"))
    out = torch.zeros(s["rows"], h, d, dtype=torch.float64, device=pk.device)
    for b in range(len(lens)):
        lo, hi = start[b], start[b + 1]
        k, v = (torch.cat([x, gather(s[n], table[b], lens[b])]).double() for x, n in ((pk, "k_pages"), (pv, "v_pages")))
        limit = p + lens[b] - (hi - lo) + torch.arange(hi - lo, device=k.device)
        hidden = torch.arange(k.shape[0], device=k.device)[None] > limit[:, None]
        for i in range(hk):
            heads = slice(i * (h // hk), (i + 1) * (h // hk))
            score = torch.einsum("tgd,kd->gtk", s["q"][lo:hi, heads].double(), k[:, i]) / d ** 0.5
            out[lo:hi, heads] = torch.einsum("gtk,kd->tgd", score.masked_fill(hidden, -torch.inf).softmax(-1), v[:, i])
    return out.reshape(s["rows"], h * d)
