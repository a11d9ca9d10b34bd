"""Speculative decoding on a quantized cache: every call of the library in one loop.

    python examples/speculative_decode.py

A small transformer of random Q8_0 weights generates for two prompts at once.  Each round drafts
a tree with its own first layer (the likeliest token of each depth, and the second likeliest
beside it), runs all layers over all nodes in one pass, verifies them against the target's
logits, and keeps the accepted path in the cache.  The same model, one token a round, is run
beside it: greedily both emit the same tokens, the first in fewer rounds.
"""
from __future__ import annotations

import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

import dyninfer_amd as d

HIDDEN, HEADS, KV_HEADS, DIM, FFN, LAYERS, VOCAB = 512, 8, 2, 64, 1024, 2, 2048
PAGE, PAGES_PER_SEQ = 16, 32  # a cache of 512 positions a sequence


def q8_0(gen, rows: int, cols: int, gain: float = 1.0) -> d.QWeight:
    """Random weights of standard deviation gain / sqrt(cols) in GGUF Q8_0 blocks."""
    n = rows * cols // 32
    blocks = torch.empty((n, 34), dtype=torch.uint8, device="cuda")
    blocks[:, :2] = torch.full((n,), gain / 73.3 / cols ** 0.5, device="cuda").half().view(torch.uint8).view(n, 2)
    blocks[:, 2:] = torch.randint(-127, 128, (n, 32), device="cuda", generator=gen).to(torch.int8).view(torch.uint8)
    return d.QWeight(d.ENC_Q8_0, rows, cols, blocks.view(-1))


def norm(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


class Model:
    def __init__(self, ctx: d.Context, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx = ctx
        self.embed = q8_0(gen, VOCAB, HIDDEN, HIDDEN ** 0.5)
        self.head = q8_0(gen, VOCAB, HIDDEN, 4.0)
        kv = KV_HEADS * DIM
        self.layers = []
        for layer in range(LAYERS):
            # the later layers change little, so the first one drafts well
            out = 1.0 if layer == 0 else 0.25
            self.layers.append(dict(
                qkv=[q8_0(gen, HEADS * DIM, HIDDEN), q8_0(gen, kv, HIDDEN), q8_0(gen, kv, HIDDEN)],
                o=q8_0(gen, HIDDEN, HEADS * DIM, out), gu=[q8_0(gen, FFN, HIDDEN), q8_0(gen, FFN, HIDDEN)],
                down=q8_0(gen, HIDDEN, FFN, out)))
        self.table = ctx.rope_table(PAGE * PAGES_PER_SEQ, DIM, theta=10000.0)

    def new_cache(self, seqs: int):
        return [d.KVCache.empty(seqs * PAGES_PER_SEQ, KV_HEADS, DIM, PAGE, d.KV_Q8, d.KV_Q8) for _ in range(LAYERS)]

    def logits(self, ids, positions, caches, batch, mask=None, layers: int = LAYERS):
        """Logits of the batch's rows; their keys and values go into the caches of `layers` layers."""
        ctx, n = self.ctx, batch.tokens
        x = ctx.embedding(self.embed, ids)
        rope = d.Rope(self.table, positions, DIM, "half")
        for w, cache in zip(self.layers[:layers], caches):
            q, k, v = ctx.qlinear_multi(w["qkv"], norm(x))
            q, k, v = q.view(n, HEADS, DIM), k.view(n, KV_HEADS, DIM), v.view(n, KV_HEADS, DIM)
            q = ctx.kv_append(cache, batch, k, v, rope=rope, q=q)
            a = ctx.tree_attention(cache, batch, q, mask=mask)
            x = x + ctx.qlinear(w["o"], a.view(n, HEADS * DIM))
            gate, up = ctx.qlinear_multi(w["gu"], norm(x))
            x = x + ctx.qlinear(w["down"], torch.nn.functional.silu(gate) * up)
        return ctx.qlinear(self.head, norm(x))


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def generate(model: Model, prompts, count: int, depth: int, temperature: float = 0.0, seed: int = 0):
    """`count` tokens after each prompt (lists of ids), with drafts of `depth` tokens (0: none).
    Returns the tokens, the rounds it took, and the logits that the last token of each round was
    chosen from."""
    ctx, seqs = model.ctx, len(prompts)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    caches = model.new_cache(seqs)
    pages = i32([[s * PAGES_PER_SEQ + p for p in range(PAGES_PER_SEQ)] for s in range(seqs)])

    # the prompts but for their last tokens, as chains
    lens = [len(p) - 1 for p in prompts]
    starts = [sum(lens[:s]) for s in range(seqs + 1)]
    ids = torch.tensor([t for p in prompts for t in p[:-1]], dtype=torch.int64, device="cuda")
    batch = d.KVBatch(pages, i32([0] * seqs), i32(starts), starts[-1], max(lens), max(lens))
    if starts[-1]:
        model.logits(ids, i32([i for n in lens for i in range(n)]), caches, batch)
    out = [[] for _ in prompts]
    last = torch.tensor([p[-1] for p in prompts], dtype=torch.int64, device="cuda")
    lengths, rounds, chosen = i32(lens), 0, []

    # a tree's shape is the same in every round: the main path and a leaf beside each of its nodes
    parents, depths = [0], [0]
    main = 0
    for step in range(1, depth + 1):
        parents += [main, main]
        depths += [step, step]
        main = len(parents) - 2
    nodes = len(parents)
    sees = []
    for i, p in enumerate(parents):
        sees.append(1 << i | (sees[p] if i else 0))
    mask = torch.tensor(sees * seqs, dtype=torch.int64, device="cuda")[:, None]
    parents_dev, depth_dev = i32(parents * seqs), i32(depths).repeat(seqs)
    tree_starts = i32([nodes * s for s in range(seqs + 1)])
    one = i32(list(range(seqs + 1)))
    temps = torch.full((seqs,), temperature, device="cuda")

    while min(len(o) for o in out) < count:
        top = int(lengths.max()) + nodes
        tokens = torch.zeros((seqs, nodes), dtype=torch.int64, device="cuda")
        tokens[:, 0] = last
        draft = last
        for step in range(depth):  # the first layer alone; its rows are written again by the full pass
            b = d.KVBatch(pages, lengths + step, one, seqs, 1, top)
            two = model.logits(draft.contiguous(), lengths + step, caches, b, layers=1).topk(2, -1).indices
            tokens[:, 1 + 2 * step:3 + 2 * step] = two
            draft = two[:, 0]
        b = d.KVBatch(pages, lengths, tree_starts, seqs * nodes, nodes, top)
        logits = model.logits(tokens.view(-1), lengths.repeat_interleave(nodes) + depth_dev, caches, b, mask=mask)
        path, counts, last = ctx.draft_verify(
            logits, tokens.view(-1), parents_dev, tree_starts, nodes, temperature=temps,
            uniform=torch.rand(seqs * nodes, device="cuda", generator=gen),
            noise=torch.empty((seqs, VOCAB), device="cuda").exponential_(generator=gen).clamp_min_(1e-30))
        for cache in caches:
            ctx.kv_commit(cache, b, path, counts)
        lengths = lengths + counts
        rounds += 1
        for s, (p, c, t) in enumerate(zip(path.tolist(), counts.tolist(), last.tolist())):
            out[s] += [int(tokens[s, i]) for i in p[1:c]] + [t]
        at = path[torch.arange(seqs, device="cuda"), (counts - 1).long()].long()
        chosen.append(logits.view(seqs, nodes, VOCAB)[torch.arange(seqs, device="cuda"), at])
    return [o[:count] for o in out], rounds, chosen


def main():
    ctx = d.Context(0)
    model = Model(ctx)
    prompts = [[5, 99, 1203, 7, 42], [17, 1999, 3]]
    for depth in (0, 4):
        generate(model, prompts, 4, depth)  # warm up
        torch.cuda.synchronize()
        t = time.perf_counter()
        tokens, rounds, _ = generate(model, prompts, 48, depth)
        t = time.perf_counter() - t
        print(f"drafts of {depth}: 48 tokens for {len(prompts)} prompts in {rounds} rounds, {1e3 * t:.1f} ms")
        for p, o in zip(prompts, tokens):
            print("  ", p, "->", o)


if __name__ == "__main__":
    main()
