"""Scoring prompts: log probabilities of their own tokens, in one pass or in chunks.

    python examples/score_prompt.py

A small transformer of random Q8_0 weights, whose query and key heads are normed, reads several
prompts of different lengths packed one after the other.  Keys and values are kept as they are
(the pass needs no cache of pages): a chunk of a prompt attends over those of the chunks before it
and its own.  Each token gets its log probability under the tokens before it, its rank, and the
likeliest alternatives.  The same keys go into a quantized cache on the way, from which the
prompts are continued one token at a time.
"""
from __future__ import annotations

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import torch

from speculative_decode import DIM, FFN, HEADS, HIDDEN, KV_HEADS, LAYERS, PAGE, PAGES_PER_SEQ, VOCAB, d, i32, norm, q8_0


class Model:
    def __init__(self, ctx: d.Context, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        weight = lambda: d.HeadNorm(1 + 0.1 * torch.randn(DIM, device="cuda", generator=gen))
        self.ctx, kv = ctx, KV_HEADS * DIM
        self.embed, self.head = q8_0(gen, VOCAB, HIDDEN, HIDDEN ** 0.5), q8_0(gen, VOCAB, HIDDEN, 4.0)
        self.layers = [dict(
            qkv=[q8_0(gen, HEADS * DIM, HIDDEN), q8_0(gen, kv, HIDDEN), q8_0(gen, kv, HIDDEN)], q_norm=weight(), k_norm=weight(),
            o=q8_0(gen, HIDDEN, HEADS * DIM), gu=[q8_0(gen, FFN, HIDDEN), q8_0(gen, FFN, HIDDEN)], down=q8_0(gen, HIDDEN, FFN))
            for _ in range(LAYERS)]
        self.table = ctx.rope_table(PAGE * PAGES_PER_SEQ, DIM, theta=10000.0)

    def run(self, ids, positions, attend):
        """Logits of the rows; attend(layer, weights, q, k, v, rope) is the attention of a layer."""
        ctx, n = self.ctx, len(ids)
        x = ctx.embedding(self.embed, ids)
        rope = d.Rope(self.table, positions, DIM, "half")
        for layer, w in enumerate(self.layers):
            q, k, v = ctx.qlinear_multi(w["qkv"], norm(x))
            a = attend(layer, w, q.view(n, HEADS, DIM), k.view(n, KV_HEADS, DIM), v.view(n, KV_HEADS, DIM), rope)
            x = x + ctx.qlinear(w["o"], a.view(n, HEADS * DIM))
            gate, up = ctx.qlinear_multi(w["gu"], norm(x))
            x = x + ctx.qlinear(w["down"], torch.nn.functional.silu(gate) * up)
        return ctx.qlinear(self.head, norm(x))


def starts_of(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths) + 1)]


def score(model: Model, prompts, chunk: int = 1 << 20, top: int = 3, caches=None, pages=None):
    """Of each prompt, for the tokens behind its first: `TokenLogprobs`; and the logits of its last row.
    `chunk` tokens of every prompt a pass.  `caches`, one a layer, take the keys and values too."""
    ctx = model.ctx
    kept = [[None] * len(prompts) for _ in range(LAYERS)]  # (keys, values) of a layer and a prompt
    scores, last = [[] for _ in prompts], [None] * len(prompts)
    for at in range(0, max(map(len, prompts)), chunk):
        parts = [p[at:at + chunk] for p in prompts]
        news, nks = [len(p) for p in parts], [min(len(p), at + chunk) for p in prompts]
        starts, n = starts_of(news), sum(news)
        batch = d.PromptBatch(i32(starts), max(news), i32(starts_of(nks)), max(nks))
        if caches:
            paged = d.KVBatch(pages, i32([m - k for m, k in zip(nks, news)]), i32(starts), n, max(news), max(nks))

        def attend(layer, w, q, k, v, rope):
            if caches:
                ctx.kv_append(caches[layer], paged, k, v, rope=rope, k_norm=w["k_norm"])
            q, k = ctx.qk_norm_rope(q, k, rope, q_norm=w["q_norm"], k_norm=w["k_norm"])
            own = kept[layer]
            for s, (a, b) in enumerate(zip(starts, starts[1:])):
                old = own[s] or (k[:0], v[:0])
                own[s] = (torch.cat([old[0], k[a:b]]), torch.cat([old[1], v[a:b]]))
            return ctx.prompt_attention(q, torch.cat([x for x, _ in own]), torch.cat([x for _, x in own]), batch)

        ids = torch.tensor([t for p in parts for t in p], dtype=torch.int64, device="cuda")
        logits = model.run(ids, i32([at + i for p in parts for i in range(len(p))]), attend)
        # a row is scored by the token behind it; the last row of a prompt has none (-1)
        behind = [t for p in prompts for t in (p[at + 1:at + chunk + 1] + [-1])[:len(p[at:at + chunk])]]
        got = ctx.token_logprobs(logits, torch.tensor(behind, dtype=torch.int64, device="cuda"), top=top)
        for s, (a, b) in enumerate(zip(starts, starts[1:])):
            if a == b:
                continue
            scores[s].append([x[a:b] for x in got])
            last[s] = logits[b - 1]
    return [d.TokenLogprobs(*[torch.cat(x)[:-1] for x in zip(*s)]) for s in scores], torch.stack(last)


def continue_from(model: Model, caches, pages, lengths, logits, count: int):
    """`count` tokens after each prompt, the likeliest ones, and their log probabilities."""
    ctx, seqs = model.ctx, len(lengths)
    one, lengths, most, out = i32(list(range(seqs + 1))), i32(lengths), max(lengths), []
    for _ in range(count):
        best = ctx.token_logprobs(logits, top=1)
        out.append((best.top_tokens[:, 0], best.top_logprobs[:, 0]))
        most += 1
        batch = d.KVBatch(pages, lengths, one, seqs, 1, most)

        def attend(layer, w, q, k, v, rope):
            q = ctx.kv_append(caches[layer], batch, k, v, rope=rope, q=q, q_norm=w["q_norm"], k_norm=w["k_norm"])
            return ctx.tree_attention(caches[layer], batch, q)

        logits = model.run(best.top_tokens[:, 0].contiguous(), lengths, attend)
        lengths = lengths + 1
    return [torch.stack(x, 1) for x in zip(*out)]


def main():
    ctx = d.Context(0)
    model = Model(ctx)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, VOCAB, (n,), generator=gen).tolist() for n in (90, 7, 41)]
    pages = i32([[s * PAGES_PER_SEQ + p for p in range(PAGES_PER_SEQ)] for s in range(len(prompts))])
    caches = [d.KVCache.empty(len(prompts) * PAGES_PER_SEQ, KV_HEADS, DIM, PAGE) for _ in range(LAYERS)]
    for chunk in (1 << 20, 32):
        scores, last = score(model, prompts, chunk, caches=caches, pages=pages)
        for p, s in zip(prompts, scores):
            print(f"chunks of {chunk}: {len(p)} tokens, {float(s.logprobs.mean()):.3f} a token, median rank {int(s.ranks.median())}")
    tokens, logp = continue_from(model, caches, pages, [len(p) for p in prompts], last, 8)
    for p, t, l in zip(prompts, tokens.tolist(), logp.tolist()):
        print("  ", p[-3:], "->", t, [round(x, 2) for x in l])


if __name__ == "__main__":
    main()
