"""A model's serving step made of the framework's operators: LlamaQ4's own layers (q4_linear, rmsnorm, embedding, lm_head) around
the batched serving operators, for sequences that share a prompt prefix and verify drafted tokens, against LlamaQ4.step on each
sequence alone."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

CFG = dict(hidden_size=1024, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2, head_dim=128,
           intermediate_size=2048, vocab_size=4096, rms_norm_eps=1e-5, rope_theta=500000.0,
           max_position_embeddings=4096, tie_word_embeddings=True, hidden_act="silu", attention_bias=False,
           initializer_range=0.02)
PREFIX, TAILS, NEW, DRAFTS, PAGE = 37, (5, 1, 20), 12, 3, 16
# Against the model's own step two values are rounded to fp16 in each of the two layers, q and the attention's output, each by at
# most 2^-11 of itself; twice that for what the layers behind make of it. Relative to the largest logit.
TOL = 2 * 2 * 2 * 2.0**-11


@pytest.fixture(scope="module")
def model():
    import q4b
    return q4b.LlamaQ4(None, group=128, max_ctx=1024, vocab_chunk=CFG["vocab_size"], sd=q4b.SyntheticStateDict(CFG, seed=5),
                       cfg=CFG, max_chunk=64)


def _alone(m, prompt):
    """Greedy tokens of one sequence by the model's own step, the logits that they came from."""
    caches = m.new_caches()
    nxt, lg = m.step(torch.from_numpy(prompt).reshape(1, -1), torch.tensor([0]), torch.tensor([len(prompt) - 1]), caches, 64)
    toks, logits = [int(nxt)], [lg[0].cpu().numpy()]
    for i in range(NEW + DRAFTS):
        nxt, lg = m.step(nxt.reshape(1, 1), torch.tensor([len(prompt) + i]), torch.tensor([0]), caches, 128)
        toks.append(int(nxt))
        logits.append(lg[0].cpu().numpy())
    return toks, logits


def _forward(m, tokens, pools, batch, prefix_len):
    """tokens [rows] -> logits [rows, V]: one step of a batch over the paged cache."""
    import q4b
    H, Hkv, hd = CFG["num_attention_heads"], CFG["num_key_value_heads"], CFG["head_dim"]
    table, lens, q_start, prefix_pages = batch
    cos, sin = m.cos[:, :hd // 2], m.sin[:, :hd // 2]
    x = m.embed.lookup(tokens)
    for ly, (kp, vp) in zip(m.layers, pools):
        qkv = ly.wqkv(q4b.rmsnorm(x, ly.ln_in, m.eps))
        q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.split([H * hd, Hkv * hd, Hkv * hd], 1))
        q = q4b.paged_rope_append(q, k, v, kp, vp, table, lens, q_start, cos, sin, prefix_len=prefix_len)
        o = q4b.prefix_attention(q, kp, vp, prefix_pages, prefix_len, table, lens, q_start)
        ly.wo(o.float(), epilogue="accumulate", out=x)
        ly.wdown(ly.wgu(q4b.rmsnorm(x, ly.ln_post, m.eps), epilogue="swiglu"), epilogue="accumulate", out=x)
    return m.embed.logits(q4b.rmsnorm(x, m.ln_f, m.eps))


def test_batched_step_equals_the_model(model):
    import q4b
    m = model
    rng = np.random.default_rng(11)
    prefix = rng.integers(0, CFG["vocab_size"], PREFIX).astype(np.int32)
    tails = [rng.integers(0, CFG["vocab_size"], n).astype(np.int32) for n in TAILS]
    want = [_alone(m, np.concatenate([prefix, t])) for t in tails]

    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)  # noqa: E731
    n_prefix, width = -(-PREFIX // PAGE), 4
    ids = rng.permutation(n_prefix + width * len(TAILS) + 2)
    prefix_pages, table = i32(ids[:n_prefix]), i32(ids[n_prefix:n_prefix + width * len(TAILS)].reshape(-1, width))
    pools = [[torch.zeros(len(ids), PAGE, CFG["num_key_value_heads"], CFG["head_dim"], dtype=torch.float16, device=DEV)
              for _ in range(2)] for _ in m.layers]

    # the prefix, once: a batch of one sequence whose own pages are the prefix's
    _forward(m, i32(prefix), pools, (prefix_pages[None], i32([PREFIX]), i32([0, PREFIX]), prefix_pages[:0]), 0)

    done = [[] for _ in TAILS]  # new tokens of each sequence
    lens = np.zeros(len(TAILS), dtype=np.int64)  # own keys
    rows = list(tails)
    compared, steps = 0, 0
    while any(len(d) < NEW for d in done):
        n = np.array([len(r) for r in rows])
        lens += n
        start = np.concatenate([[0], np.cumsum(n)])
        tokens = i32(np.concatenate(rows))
        logits = _forward(m, tokens, pools, (table, i32(lens), i32(start), prefix_pages), PREFIX)
        first = steps == 0  # the tails: one new token each, of the last row; then the last token and its drafts
        got = logits.cpu().numpy()
        choice = got.argmax(1)
        for b, (toks, ref) in enumerate(want):
            for j in ([n[b] - 1] if first else range(n[b])):
                at = len(done[b]) + (0 if first else j)
                # rows behind a wrong draft belong to no real continuation
                if not first and list(rows[b][1:j + 1]) != toks[at - j:at]:
                    choice[start[b] + j] = 0
                    continue
                top = np.abs(ref[at]).max()
                assert np.abs(got[start[b] + j] - ref[at]).max() <= TOL * top, (b, at)
                second, best = np.sort(ref[at])[-2:]
                if best - second > 2 * TOL * top:
                    assert choice[start[b] + j] == toks[at], (b, at)
                    compared += 1
                choice[start[b] + j] = toks[at]
        if first:
            new = [[int(choice[start[b + 1] - 1])] for b in range(len(TAILS))]
        else:
            target = torch.zeros(len(choice), CFG["vocab_size"], device=DEV)
            target[torch.arange(len(choice)), torch.from_numpy(choice).to(DEV)] = 1.0
            out, kept = q4b.verify_drafts(target, None, tokens, torch.full((len(choice),), 0.5, device=DEV), i32(start))
            out, kept = out.cpu().numpy(), kept.cpu().numpy()
            made = np.where(n > 0, kept + 1, 0)
            new = [out[start[b]:start[b] + made[b]].tolist() for b in range(len(TAILS))]
            lens -= n - made  # the rejected drafts' slots are written over by the next append
        rows = []
        for b, (toks, _) in enumerate(want):
            done[b] += new[b]
            assert done[b] == toks[:len(done[b])], b
            if len(done[b]) >= NEW:  # a sequence that is done has no rows
                rows.append(np.zeros(0, dtype=np.int32))
                continue
            drafts = toks[len(done[b]):len(done[b]) + DRAFTS]
            wrong = (steps + b) % (DRAFTS + 1)
            if wrong < len(drafts):
                drafts[wrong] = (drafts[wrong] + 1) % CFG["vocab_size"]
            rows.append(np.array([done[b][-1]] + drafts, dtype=np.int32))
        steps += 1
    assert compared >= 2 * NEW and steps < 2 * NEW
    assert q4b.lib().q4b_device_status(1) == 0
