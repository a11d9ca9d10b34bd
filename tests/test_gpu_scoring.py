"""The calls around prompts together, as a program uses them: norms and rotation, attention and log
probabilities one after the other against 64 bits; the same rows through the quantized cache; several
streams, and a graph; the example.

Errors of a chain: a query off by tq and a key off by tk (the norms' tolerance) move a score by
scale (tq |k| + |q| tk + tq tk) beside what the attention itself leaves; log probabilities move by
at most twice what the largest move of a logit of the row is, the entropy H by that times
sum p |ln p + H| <= 2 H."""
import importlib.util
import os
import sys

import numpy as np
import pytest
import torch

import dyninfer_amd as d
import kvref
from test_gpu_kvcache import DT, dev, i32
from test_gpu_norm_rope import HALF_STEP, normed, turned
from test_gpu_prompt import P_STEP, Prompts

pytestmark = pytest.mark.gpu

EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples")
U = 2.0**-24


class Chain:
    """Packed prompts of one layer and the scores of their rows: 4 query heads on 2 of keys."""

    def __init__(self, seed, news, dim, io, layout):
        rng = np.random.default_rng(seed)
        self.news, self.dim, self.io, self.layout = news, dim, io, layout
        self.starts = np.concatenate([[0], np.cumsum(news)]).astype(int)
        t = self.t = int(self.starts[-1])
        self.fused = dev(rng.normal(0, 1, (t, 8, dim)), DT[io])  # a product's output: queries, keys, values
        self.w = [dev(rng.normal(1, 0.3, dim).astype(np.float32)) for _ in range(2)]
        self.positions = i32(np.concatenate([np.arange(n) for n in news]))
        self.table = kvref.table(max(news), dim).astype(np.float32)
        self.rope = d.Rope(dev(self.table), self.positions, dim, layout)
        self.tokens = dev(rng.integers(0, 4 * dim, t), torch.int64)
        self.batch = d.PromptBatch(i32(self.starts), max(news))

    def run(self, ctx):
        f = self.fused
        q, k = ctx.qk_norm_rope(f[:, :4], f[:, 4:6], self.rope, d.HeadNorm(self.w[0]), d.HeadNorm(self.w[1]))
        a = ctx.prompt_attention(q, k, f[:, 6:], self.batch) * 8.0  # exact
        return ctx.token_logprobs(a.view(self.t, 4 * self.dim), self.tokens, top=4)

    def expect(self):
        """(log probabilities of all tokens, tolerance, entropy, tolerance) of every row in 64 bits."""
        f, dim, io = self.fused.double().cpu().numpy(), self.dim, self.io
        pos, out, tol = self.positions.cpu().numpy(), np.zeros((self.t, 4, dim)), np.zeros((self.t, 4, dim))
        qk = []
        for x, w in ((f[:, :4], self.w[0]), (f[:, 4:6], self.w[1])):
            want, size = turned(normed(x, w.cpu().numpy(), np.float32(1e-6), 0.0), self.table, pos, dim, self.layout == "half")
            qk.append((want, 16 * U * size + HALF_STEP[io] * np.abs(want)))
        (q, tq), (k, tk) = qk
        for a, b in zip(self.starts, self.starts[1:]):
            for h in range(4):
                x, tx, y, ty, v = q[a:b, h], tq[a:b, h], k[a:b, h // 2], tk[a:b, h // 2], f[a:b, 6 + h // 2]
                see = np.tril(np.ones((b - a, b - a), bool))
                scale = dim**-0.5
                s = np.where(see, x @ y.T * scale, -np.inf)
                # of moved inputs, and of the attention itself
                move = scale * (tx @ np.abs(y).T + np.abs(x) @ ty.T + tx @ ty.T)
                own = U * (dim + 16) * scale * (np.abs(x) + tx) @ (np.abs(y) + ty).T
                ds = np.where(see, move + own, 0).max(-1)
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out[a:b, h] = p @ v
                # e^(2 ds) - 1, and not 2 ds alone: bf16 moves scores by percents
                rel = np.expm1(2 * ds) + P_STEP[io] * np.exp(2 * ds) + U * (32 + (b - a) / 4)
                tol[a:b, h] = rel[:, None] * (p @ np.abs(v)) * (1 + HALF_STEP[io]) + HALF_STEP[io] * np.abs(out[a:b, h])
        x, dx = 8 * out.reshape(self.t, -1), 8 * tol.reshape(self.t, -1).max(-1)
        m = x.max(-1, keepdims=True)
        z = np.log(np.exp(x - m).sum(-1, keepdims=True))
        logp = x - m - z
        h = -(np.exp(logp) * logp).sum(-1)
        own = U * (64 + 8 * (np.abs(x - m) + np.abs(logp)))  # of the log probabilities on exact logits
        return logp, 2 * dx[:, None] + own, h, (2 * h * dx + 4 * dx * dx) + U * 200 * (1 + h)

    def check(self, got):
        logp, tol, h, tol_h = self.expect()
        t, r = self.tokens.cpu().numpy(), np.arange(self.t)
        lp, ranks, en, tt, tl = [x.cpu().numpy() for x in got]
        assert (np.abs(lp - logp[r, t]) <= tol[r, t]).all(), (np.abs(lp - logp[r, t]) / tol[r, t]).max()
        assert (np.abs(en - h) <= tol_h).all(), (np.abs(en - h) / tol_h).max()
        # ranks lie between the counts of tokens that are surely and that may be likelier
        mine = logp[r, t][:, None]
        slack = tol + tol[r, t][:, None]
        assert (ranks >= (logp > mine + slack).sum(-1)).all() and (ranks <= (logp > mine - slack).sum(-1)).all()
        for i in range(4):
            assert (np.abs(tl[:, i] - logp[r, tt[:, i]]) <= tol[r, tt[:, i]]).all()
            assert (ranks == i)[tt[:, i] == t].all()
        assert (np.diff(tl, axis=1) <= 0).all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dim,layout", [(64, "half"), (96, "interleaved"), (128, "half"), (256, "interleaved")])
@pytest.mark.parametrize("news", [[1], [5, 1, 40], [129, 70]])
def test_chain(ctx, io, dim, layout, news):
    c = Chain(dim + sum(news), news, dim, io, layout)
    c.check(c.run(ctx))


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_chain_in_a_graph(ctx, io):
    c = Chain(11, [33, 1, 90], 128, io, "half")
    other = Chain(12, [33, 1, 90], 128, io, "half")
    want = [[x.clone() for x in y.run(ctx)] for y in (c, other)]
    inputs = [y.fused.clone() for y in (c, other)], [y.tokens.clone() for y in (c, other)], [[w.clone() for w in y.w] for y in (c, other)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run(ctx)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = c.run(ctx)
    for turn in (1, 0, 1, 1, 0):
        c.fused.copy_(inputs[0][turn])
        c.tokens.copy_(inputs[1][turn])
        for w, x in zip(c.w, inputs[2][turn]):
            w.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[turn]):
            assert torch.equal(a, b)
        other.run(ctx)  # eager work between the replays


def test_two_streams_at_once(ctx):
    """Calls with workspaces of their own on two streams: each the same as alone."""
    cases = [Prompts(s, [3, 1], [5000 + s, 4000], 2, 4, 128, "bf16") for s in (1, 2)]
    alone = [p.run(ctx) for p in cases]
    logits = [torch.randn(5, 40000, device="cuda") for _ in cases]
    scores = [ctx.token_logprobs(x, top=5) for x in logits]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    batches = [p.batch() for p in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(6):
        for i, (p, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append((ctx.prompt_attention(p.q, p.k, p.v, batches[i]), ctx.token_logprobs(logits[i], top=5)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, l in got[i]:
            assert torch.equal(a, alone[i][0])
            assert torch.equal(l.entropy, scores[i].entropy) and torch.equal(l.top_tokens, scores[i].top_tokens)


@pytest.mark.parametrize("dim,kb,vb", [(64, d.KV_Q8, d.KV_Q4), (128, d.KV_Q8, d.KV_Q8), (256, d.KV_Q4, d.KV_Q8)])
def test_cache_and_prompt_agree(ctx, dim, kb, vb):
    """What the cache holds, read back and attended to as a prompt, and through its pages: f32
    queries of the cache's attention are two f16 terms, 2^-22 of a row's largest."""
    news, page, pages = [70, 1, 33], 16, 5
    p = Prompts(dim, news, [0] * 3, 2, 3, dim, "f32")
    rng = np.random.default_rng(5)
    cache = d.KVCache.empty(3 * pages, 2, dim, page, kb, vb)
    order = rng.permutation(3 * pages).reshape(3, pages)
    batch = d.KVBatch(i32(order), i32([0] * 3), i32(p.starts), sum(news), max(news), max(news))
    rope = d.Rope(ctx.rope_table(128, dim), i32(np.concatenate([np.arange(n) for n in news])), dim, "half")
    norms = [d.HeadNorm(dev(rng.normal(1, 0.3, dim).astype(np.float32))) for _ in range(2)]
    q = ctx.kv_append(cache, batch, p.k, p.v, rope=rope, q=p.q, q_norm=norms[0], k_norm=norms[1])
    assert torch.equal(q, ctx.qk_norm_rope(p.q, None, rope, q_norm=norms[0])[0])
    p.q = q
    p.k, p.v = ctx.kv_read(cache, batch)
    got = p.run(ctx)
    p.check(got)
    lse = torch.empty(sum(news), 6, device="cuda")
    paged = ctx.tree_attention(cache, batch, q, lse=lse)
    scale = dim**-0.5
    out, want, tol, ltol = p.expect(scale)
    ds = 2.0**-22 * scale * q.double().abs().amax(-1) * float(p.k.double().abs().sum(-1).max())
    assert ((paged.double() - out).abs() <= tol + ((2 * ds + 2.0**-23) * float(p.v.abs().max()))[..., None]).all()
    assert ((lse.double() - want).abs() <= ltol + ds + 2.0**-22 * (1 + want.abs())).all()


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("score_prompt", os.path.join(EXAMPLES, "score_prompt.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    yield mod
    sys.path.remove(EXAMPLES)


def test_example(ctx, example):
    model = example.Model(ctx)
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, example.VOCAB, n).tolist() for n in (90, 2, 41, 33)]
    pages = i32(np.arange(4 * example.PAGES_PER_SEQ).reshape(4, -1))
    caches = [d.KVCache.empty(4 * example.PAGES_PER_SEQ, example.KV_HEADS, example.DIM, example.PAGE) for _ in range(example.LAYERS)]
    for chunk in (1000, 32, 7):
        scores, last = example.score(model, prompts, chunk, caches=caches, pages=pages)
        for p, s in zip(prompts, scores):
            assert s.logprobs.shape == s.ranks.shape == s.entropy.shape == (len(p) - 1,) and s.top_tokens.shape == (len(p) - 1, 3)
            assert torch.isfinite(s.logprobs).all() and (s.logprobs <= 0).all() and (s.entropy >= 0).all()
            first = s.top_tokens[:, 0] == torch.tensor(p[1:], device="cuda")
            assert torch.equal(first, s.ranks == 0)
            assert (s.top_logprobs[:, 0] >= s.logprobs).all()
        again = example.score(model, prompts, chunk)[0]
        assert all(torch.equal(a.logprobs, b.logprobs) for a, b in zip(scores, again))
        tokens, logp = example.continue_from(model, caches, pages, [len(p) for p in prompts], last, 5)
        assert tokens.shape == (4, 5) and torch.isfinite(logp).all() and (logp <= 0).all()
