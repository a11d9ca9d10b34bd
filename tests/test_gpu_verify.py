"""Verification of drafted tokens on the GPU, against the rule in 64 bits.  Outputs are whole
numbers and equal; cases in which 64 bits find a comparison closer than f32 sums can tell
(2^-16 of its sides) would be ambiguous, and the fixed seeds here hold none."""
import numpy as np
import pytest
import torch

import kvref
from test_gpu_attention import random_tree
from test_gpu_kvcache import bad, dev, i32

pytestmark = pytest.mark.gpu


class Draft:
    def __init__(self, seed, news, vocab, probs, tree=True, sharp=2.0, near=0.7):
        rng = self.rng = np.random.default_rng(seed)
        self.news, self.vocab = news, vocab
        self.starts = np.concatenate([[0], np.cumsum(news)])
        n = sum(news)
        self.parents = np.concatenate([random_tree(rng, k) if tree else np.arange(-1, k - 1) for k in news if k]).astype(int)
        self.logits = (rng.normal(0, sharp, (n, vocab))).astype(np.float32)
        close = self.logits + rng.normal(0, near, (n, vocab))
        e = np.exp(close - close.max(-1, keepdims=True))
        q = (e / e.sum(-1, keepdims=True)).astype(np.float32)
        self.tokens = np.zeros(n, np.int64)
        for b, k in enumerate(news):
            for i in range(1, k):
                row = self.starts[b] + i
                p = q[self.starts[b] + max(self.parents[row], 0)].astype(np.float64)
                self.tokens[row] = rng.choice(vocab, p=p / p.sum())
        self.probs = q if probs else None
        self.uniform = rng.random(n).astype(np.float32)
        self.noise = rng.exponential(1, (len(news), vocab)).astype(np.float32)
        self.temperature = np.where(rng.random(len(news)) < 0.25, 0, rng.uniform(0.5, 1.5, len(news))).astype(np.float32)

    def run(self, ctx, dtype=torch.float32, pdtype=torch.float32, **kw):
        logits = kw.pop("logits", None)
        logits = dev(self.logits, dtype) if logits is None else logits
        width = max(self.news)
        got = ctx.draft_verify(logits, dev(self.tokens), i32(self.parents), i32(self.starts), width,
                               uniform=dev(self.uniform), noise=dev(self.noise), temperature=dev(self.temperature),
                               draft_probs=None if self.probs is None else dev(self.probs, pdtype), **kw)
        torch.cuda.synchronize()
        return got

    def expect(self, dtype=torch.float32, pdtype=torch.float32):
        cast = lambda a, t: dev(a, t).float().cpu().numpy()
        logits = cast(self.logits, dtype)
        probs = None if self.probs is None else cast(self.probs, pdtype)
        path = np.full((len(self.news), max(self.news)), -1)
        counts, token = [], []
        for b, k in enumerate(self.news):
            r = slice(self.starts[b], self.starts[b] + k)
            if k == 0:
                counts.append(0), token.append(-1)
                continue
            p, t = kvref.verify(logits[r], self.tokens[r], self.parents[r], self.temperature[b], self.uniform[r],
                                self.noise[b], None if probs is None else probs[r])
            path[b, :len(p)] = p
            counts.append(len(p)), token.append(t)
        return path, counts, token

    def check(self, ctx, dtype=torch.float32, pdtype=torch.float32, **kw):
        path, counts, token = (x.cpu().numpy() for x in self.run(ctx, dtype, pdtype, **kw))
        want = self.expect(dtype, pdtype)
        assert np.array_equal(path, want[0])
        assert np.array_equal(counts, want[1]) and np.array_equal(token, want[2])
        return path, counts, token


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 7, 32, 501, 16384, 16391, 40001])
def test_against_the_rule(ctx, probs, tree, dtype, vocab):
    news = [1, 5, 0, 9, 2, 16, 7, 3]
    accepted = 0
    for seed in range(4):
        dr = Draft(seed + vocab, news, vocab, probs, tree)
        accepted += dr.check(ctx, dtype, torch.bfloat16 if seed % 2 else torch.float32)[1].sum()
    assert accepted > 4 * 7 or not probs  # more than the roots


@pytest.mark.parametrize("probs", [False, True])
def test_many_siblings(ctx, probs):
    """Star-shaped trees with poor drafts: what is left after several rejections at one node."""
    rejected = 0
    for seed in range(20):
        dr = Draft(100 + seed, [12, 12, 12], 60, probs, near=3.0)
        dr.parents[:] = np.tile([-1] + [0] * 11, 3)
        dr.temperature[:] = 1
        if not probs:
            dr.tokens[1:12] = np.argsort(-dr.logits[0])[:11]      # the likeliest: little is left
            dr.tokens[13:24] = dr.tokens[13]                       # one token over and over
        path, _, _ = dr.check(ctx)
        rejected += (path[:, 1] != 1).sum()
    assert rejected > 5


def test_next_token_follows_the_target(ctx):
    """Chains of one draft: emitted tokens are distributed as the target, whatever the draft."""
    n, vocab = 4000, 6
    rng = np.random.default_rng(0)
    logit = rng.normal(0, 1, vocab).astype(np.float32)
    p = np.exp(logit) / np.exp(logit).sum()
    q = np.exp(rng.normal(0, 1, vocab))
    q = (q / q.sum()).astype(np.float32)
    dr = Draft(3, [2] * n, vocab, True)
    dr.logits[:] = logit
    dr.probs[:] = q
    dr.temperature[:] = 1
    dr.parents = np.tile([-1, 0], n)
    dr.tokens = rng.choice(vocab, size=2 * n, p=q.astype(np.float64) / q.astype(np.float64).sum())
    path, counts, token = (x.cpu().numpy() for x in dr.run(ctx))
    first = np.where(counts == 2, dr.tokens[1::2], token)
    seen = np.bincount(first, minlength=vocab) / n
    assert np.abs(seen - p).max() <= 5 * np.sqrt(0.25 / n)  # five standard deviations


def test_special_logits(ctx):
    """-inf, +inf, NaN, ties, and rows of -inf only."""
    vocab = 40
    dr = Draft(7, [3] * 8, vocab, False, tree=False)
    x = dr.logits
    inf, nan = np.inf, np.nan
    x[0] = -inf                      # nothing: no child, no token
    x[3, :] = nan
    x[6, 5:9] = inf                  # four tokens share all of it
    x[9, ::2] = nan
    x[12, :20] = -inf
    x[15, [11, 30]] = 50.0           # a tie of the largest
    x[18, :] = -3.4e38
    x[21, [3, 4]] = [3.4e38, -3.4e38]
    dr.temperature[:] = [1, 1, 1, 0.7, 1, 0, 0, 1]
    dr.tokens[[7, 10, 13, 16, 19, 22]] = [6, 1, 25, 11, 0, 3]
    dr.uniform[[7, 10, 13, 16, 19, 22]] = [0.2, 0.001, 0.001, 0.5, 0.5, 0.5]
    path, counts, token = dr.check(ctx)
    assert token[0] == -1 and token[1] == -1 and counts[0] == 1 and counts[2] >= 2 and counts[5] >= 2


def test_tokens_and_parents_out_of_range(ctx):
    dr = Draft(8, [6, 6], 100, False, tree=False)
    dr.temperature[:] = [1.0, 0.0]
    dr.tokens[1], dr.tokens[7] = 100, -1
    path, counts, _ = dr.check(ctx)
    assert (counts == 1).all()
    dr = Draft(9, [6, 6], 100, True, tree=False)
    dr.parents[:] = [-1, 5, 99, 2, -3, 4] * 2
    assert (dr.check(ctx)[1] == 1).all()


def test_everything_rejected_away(ctx):
    """Drafts equal to the target leave nothing to draw from: the target itself is drawn from."""
    dr = Draft(10, [4, 4], 5, True)
    dr.parents[:] = [-1, 0, 0, 0] * 2
    dr.logits[:] = 0
    dr.probs[:] = 0.25                # more than the target's 0.2 everywhere
    dr.uniform[:] = 0.9
    dr.temperature[:] = 1
    path, counts, token = dr.check(ctx)
    assert (counts == 1).all() and (token == dr.noise.argmin(-1)).all()


def test_strides_stream_graph_and_chains(ctx):
    dr = Draft(11, [4, 6, 1], 1001, True, tree=False)
    dr.temperature[:] = 1
    want = dr.check(ctx)
    wide = torch.full((sum(dr.news), 1008), float("nan"), device="cuda")
    wide[:, 3:1004] = dev(dr.logits)
    dr.check(ctx, logits=wide[:, 3:1004])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    dr.check(ctx, stream=s)
    args = (dev(dr.logits), dev(dr.tokens), None, i32(dr.starts), 6)  # chains without parents, temperature 1
    kw = dict(uniform=dev(dr.uniform), noise=dev(dr.noise), draft_probs=dev(dr.probs))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ctx.draft_verify(*args, **kw)
    for _ in range(3):
        for t in got:
            t.fill_(77)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(got, want))


def test_refusals(ctx):
    dr = Draft(12, [3, 2], 64, True)
    logits, tok, par, st = dev(dr.logits), dev(dr.tokens), i32(dr.parents), i32(dr.starts)
    kw = dict(uniform=dev(dr.uniform), noise=dev(dr.noise), temperature=dev(dr.temperature), draft_probs=dev(dr.probs))
    run = lambda l=logits, t=tok, p=par, s=st, m=3, **o: ctx.draft_verify(l, t, p, s, m, **{**kw, **o})
    run()
    bad(lambda: run(l=logits.cpu()))
    bad(lambda: run(l=logits.half()), 2)
    bad(lambda: run(l=logits.T.contiguous().T))
    bad(lambda: run(l=logits[:1].expand(5, 64)))
    bad(lambda: run(t=tok.int()))
    bad(lambda: run(t=tok[:3]))
    bad(lambda: run(p=par.long()))
    bad(lambda: run(s=st.cpu()))
    bad(lambda: run(m=6))
    bad(lambda: run(uniform=kw["uniform"].double()))
    bad(lambda: run(noise=kw["noise"][:1]))
    bad(lambda: run(noise=kw["noise"].bfloat16()))
    bad(lambda: run(temperature=kw["temperature"][:1]))
    bad(lambda: run(draft_probs=kw["draft_probs"][:2]))
    bad(lambda: run(draft_probs=kw["draft_probs"].half()), 2)
    bad(lambda: run(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()


def test_infinite_temperature(ctx):
    """Every token of a logit above -inf is as likely: the smallest noise among them is drawn."""
    c = Draft(70, [1] * 40, 1003, False)
    c.logits[c.rng.random(c.logits.shape) < 0.5] = -np.inf
    c.temperature[:] = np.inf
    _, _, token = c.run(ctx)
    want = np.where(np.isinf(c.logits), np.inf, c.noise).argmin(-1)
    assert (token.cpu().numpy() == want).all()


@pytest.mark.parametrize("vocab", [4096, 4099, 20008])
@pytest.mark.parametrize("dtype,pdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)])
def test_siblings_after_rejections(ctx, vocab, dtype, pdtype):
    """Drafts far from the target, so that rejections at a node sum its row, of whole eights and not."""
    c = Draft(71 + vocab, [16, 9, 1, 16, 12, 16], vocab, True, near=2.5)
    c.temperature[:] = 1.0
    c.check(ctx, dtype, pdtype)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("tokens", [0, 3])
def test_rounds_without_rows(ctx, tokens, probs):
    """Sequences of which none has rows in the call (or may have any): count 0 and no token."""
    vocab = 40
    logits = torch.zeros((tokens, vocab), device="cuda")
    path, counts, token = ctx.draft_verify(
        logits, torch.zeros(tokens, dtype=torch.int64, device="cuda"), None, i32([0, 0, tokens, tokens]), 0,
        uniform=torch.zeros(tokens, device="cuda"), noise=torch.ones((3, vocab), device="cuda"),
        temperature=torch.tensor([1.0, 0.0, 1.0], device="cuda"), draft_probs=logits if probs else None)
    assert path.shape == (3, 0) and counts.tolist() == [0, 0, 0] and token.tolist() == [-1, -1, -1]


def test_too_many_sequences(ctx):
    """A launch's threads are counted in 32 bits."""
    n = 1 << 22
    bad(lambda: ctx.draft_verify(torch.zeros((1, 1), device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), None,
                                 torch.zeros(n + 1, dtype=torch.int32, device="cuda"), 1,
                                 uniform=torch.zeros(1, device="cuda"), noise=torch.ones((n, 1), device="cuda")), 2)


def decidable(dr, dtype=torch.float32, pdtype=torch.float32):
    """How far the closest decision of a Draft is from a tie, in 64 bits: the smallest of the
    differences u q - R(c) at the children tried and of the largest two scores at the end, each
    over what its f32 error scales with.  R_k = max(p - a q, 0) / w: p and a q are rounded on their own,
    and w, a sum of such, is off by a part of 1."""
    cast = lambda a, t: torch.from_numpy(a).to(t).double().numpy()
    logits = cast(dr.logits, dtype)
    probs = None if dr.probs is None else cast(dr.probs, pdtype)
    least = np.inf
    for b, n in enumerate(dr.news):
        t = float(dr.temperature[b])
        if n == 0 or not t > 0:
            continue
        r0, cur, a, w, gone = dr.starts[b], 0, 0.0, 1.0, []

        def p_of(node):
            e = np.exp((logits[r0 + node] - logits[r0 + node].max()) / t)
            return e / e.sum()

        def rest():
            if probs is not None:
                return np.maximum(p - a * probs[r0 + cur], 0)
            left = p.copy()
            left[gone] = 0
            return left

        p = p_of(0)
        for i in range(1, n):
            if dr.parents[r0 + i] != cur:
                continue
            tok, u = dr.tokens[r0 + i], float(dr.uniform[r0 + i])
            q = 1.0 if probs is None else probs[r0 + cur, tok]
            side = rest()[tok] / w
            err = (p[tok] + (0 if probs is None else a * q)) / w + side / w + u * q
            least = min(least, abs(u * q - side) / err if u * q or side else 1.0)
            if u * q < side:
                cur, a, w, gone, p = i, 0.0, 1.0, [], p_of(i)
            elif probs is not None:
                a += w
                w = rest().sum()
                assert w > 0  # a case of its own
            else:
                gone.append(tok)
                w = rest().sum()
        aq = 0 if probs is None else a * probs[r0 + cur]
        score, err = rest() / dr.noise[b], (p + aq) / dr.noise[b]
        top = score.argmax()
        others = np.arange(dr.vocab) != top
        if others.any():
            least = min(least, ((score[top] - score) / (err[top] + err))[others].min())
    return least


def check_decidable(dr, ctx, dtype=torch.float32, pdtype=torch.float32):
    assert decidable(dr, dtype, pdtype) > 2.0 ** -16
    return dr.check(ctx, dtype, pdtype)


LARGE_TREES = [(64, False, 200), (64, True, 210), (64, True, 220), (300, False, 200), (300, True, 205), (300, True, 210)]


def large_trees(vocab, probs, seed):
    """Trees of more nodes than the walk holds at a time, whose nodes have children far behind them."""
    dr = Draft(seed, [600, 257, 256, 1, 513], vocab, probs, near=1.5)
    for b, n in enumerate(dr.news):
        for i in range(1, n):
            # some hang on the root, before the boundary and behind it, the others on any node
            up = 0 if dr.rng.random() < (1 / 30 if i < 256 else 1 / 8) else int(dr.rng.integers(0, i))
            dr.parents[dr.starts[b] + i] = up
            p = (dr.probs if probs else np.exp(dr.logits))[dr.starts[b] + up].astype(np.float64)
            dr.tokens[dr.starts[b] + i] = dr.rng.choice(vocab, p=p / p.sum())
            u = dr.uniform[dr.starts[b] + i]
            dr.uniform[dr.starts[b] + i] = 0.97 + 0.03 * u if i < 256 else 0.2 * u  # mostly rejected, mostly accepted
    dr.temperature[:] = 1
    return dr


@pytest.mark.parametrize("vocab,probs,seed", LARGE_TREES)
def test_trees_of_more_nodes_than_the_walk_holds(ctx, vocab, probs, seed):
    """Rejections at a node before the boundary go on to its children behind it."""
    dr = large_trees(vocab, probs, seed)
    path, counts, _ = check_decidable(dr, ctx)
    assert any((p[:c] > 256).any() for p, c in zip(path, counts))  # from one group of nodes to the next


def long_chains(probs):
    """Chains that are accepted past the boundary."""
    dr = Draft(300, [700, 300, 257], 40, probs, tree=False, near=0.05)
    dr.uniform *= 0.3
    dr.temperature[:] = [1, 0, 1]
    n0, n1 = dr.starts[1], dr.starts[2]
    best = dr.logits.argmax(-1)
    dr.tokens[n0 + 1:n1] = best[n0:n1 - 1]  # greedy: all accepted
    for b in (0, 2):
        dr.tokens[dr.starts[b] + 1:dr.starts[b + 1]] = best[dr.starts[b]:dr.starts[b + 1] - 1]
        if not probs:
            dr.logits[np.arange(dr.starts[b], dr.starts[b + 1]), best[dr.starts[b]:dr.starts[b + 1]]] += 4
    return dr


@pytest.mark.parametrize("probs", [False, True])
def test_chains_of_more_nodes_than_the_walk_holds(ctx, probs):
    dr = long_chains(probs)
    _, counts, _ = check_decidable(dr, ctx)
    assert counts[1] == 300


LARGE_PIECES = [(20001, torch.float32, 400), (32768, torch.bfloat16, 401), (40001, torch.float32, 402), (40001, torch.bfloat16, 403)]


def large_pieces(vocab, probs, seed):
    return Draft(seed, [8] * 60 + [1, 37, 0, 6], vocab, probs)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("vocab,dtype,seed", LARGE_PIECES)
def test_many_rows_of_several_pieces(ctx, vocab, dtype, seed, probs):
    """Rows so many that the statistics take them 16384 logits at a time, the last piece shorter."""
    check_decidable(large_pieces(vocab, probs, seed), ctx, dtype)
