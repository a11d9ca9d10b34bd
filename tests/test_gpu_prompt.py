"""Causal attention of packed prompts on the GPU, against 64 bits.

Tolerance of an output, from what is rounded: a score is a sum of d exact or once rounded products
in f32, off by ds = 2^-24 (d + 16) scale sum |q k| (its factor, the difference and the exponential
lie within the 16); it moves a probability by ds of itself and the sum of all by as much.  A
probability is rounded once to bf16 before the product with v (2^-8), in f32 not; the sums over
L keys of p and p v are f32, joined from 32-key pieces: 2^-24 (32 + L / 4).  Then half a step of
the output's type.  Log-sum-exp: ds, its own sum and its own two roundings."""
import numpy as np
import pytest
import torch

import dyninfer_amd as d
from test_gpu_kvcache import DT, HOW, i32, rows

pytestmark = pytest.mark.gpu

HALF_STEP = {"f32": 2.0**-24, "bf16": 2.0**-8}
P_STEP = {"f32": 0.0, "bf16": 2.0**-8}


class Prompts:
    def __init__(self, seed, news, priors, kv_heads, group, dim, io, how=0, spare=0, key_spare=0):
        rng = self.rng = np.random.default_rng(seed)
        self.news, self.nks, self.group, self.dim, self.io = news, [n + p for n, p in zip(news, priors)], group, dim, io
        self.starts = np.concatenate([[0], np.cumsum(news)]).astype(int)
        self.key_starts = np.concatenate([[0], np.cumsum(self.nks)]).astype(int)
        t, k = int(self.starts[-1]) + spare, int(self.key_starts[-1]) + key_spare
        self.q, _ = rows(rng, t, kv_heads * group, dim, DT[io], HOW[how % 4])
        self.k, _ = rows(rng, k, kv_heads, dim, DT[io], HOW[(how + 1) % 4])
        self.v, _ = rows(rng, k, kv_heads, dim, DT[io], HOW[(how + 2) % 4])
        self.own_keys = any(priors) or key_spare != spare
        self.kv_heads = kv_heads

    def batch(self, max_new=None, max_keys=None):
        return d.PromptBatch(i32(self.starts), max(self.news) if max_new is None else max_new,
                             i32(self.key_starts) if self.own_keys else None,
                             max(max(self.nks), 0) if max_keys is None else max_keys)

    def run(self, ctx, **kw):
        lse = torch.full((self.q.shape[0], self.q.shape[1]), 7.0, device="cuda")
        batch = kw.pop("batch", None) or self.batch()
        out = ctx.prompt_attention(self.q, self.k, self.v, batch, lse=lse, **kw)
        torch.cuda.synchronize()
        return out, lse

    def expect(self, scale, most=None):
        """(out, lse, tolerance of each) in 64 bits, NaN in rows the call leaves out."""
        t, h = self.q.shape[:2]
        q, k, v = (x.double().contiguous() for x in (self.q, self.k, self.v))
        out = torch.full((t, h, self.dim), float("nan"), dtype=torch.float64, device="cuda")
        lse = torch.full((t, h), float("nan"), dtype=torch.float64, device="cuda")
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        for b, (n, nk) in enumerate(zip(self.news, self.nks)):
            r = slice(self.starts[b], self.starts[b] + min(n, n if most is None else most))
            if r.start == r.stop:
                continue
            kr = slice(self.key_starts[b], self.key_starts[b] + nk)
            pos = torch.arange(r.stop - r.start, device="cuda") + nk - n
            see = torch.arange(nk, device="cuda")[None] <= pos[:, None]
            for x in range(h):
                kk, vv = k[kr, x // self.group], v[kr, x // self.group]
                s = q[r, x] @ kk.T.contiguous() * scale
                size = q[r, x].abs() @ kk.abs().T.contiguous() * abs(scale)
                ds = 2.0**-24 * (self.dim + 16) * torch.where(see, size, 0).amax(-1) if nk else torch.zeros(len(s), device="cuda").double()
                s = s.masked_fill(~see, float("-inf"))
                z = torch.logsumexp(s, -1) if nk else torch.full((len(s),), float("-inf"), device="cuda").double()
                p = torch.exp(s - torch.where(z == float("-inf"), 0, z)[:, None])
                o = torch.where(p[:, :, None] > 0, p[:, :, None] * vv[None], 0).sum(1) if not torch.isfinite(vv).all() else p @ vv
                sums = 2.0**-24 * (32 + nk / 4)
                out[r, x], lse[r, x] = o, z
                tol[r, x] = ((2 * ds + P_STEP[self.io] + sums)[:, None]) * (p @ vv.abs().nan_to_num(0, 0, 0)) + HALF_STEP[self.io] * o.abs() + 1e-40
                ltol[r, x] = ds + sums + 2.0**-23 * z.abs().nan_to_num(0, 0, 0) + 2.0**-23
        return out, lse, tol, ltol

    def check(self, got, scale=None, most=None, spoiled=None):
        scale = self.dim**-0.5 if scale is None else scale
        out, lse, tol, ltol = self.expect(scale, most)
        y, z = got[0].double(), got[1].double()
        mine = ~torch.isnan(lse)
        assert not torch.isnan(y[mine]).any()
        e = ((y - out).abs() / tol)[mine]
        assert (e <= 1).all(), e.max()
        assert torch.equal(z[mine] == float("-inf"), lse[mine] == float("-inf"))
        fine = mine & (lse > float("-inf"))
        e = ((z - lse).abs() / ltol)[fine]
        assert (e <= 1).all(), e.max()
        assert (got[0][mine & ~fine] == 0).all()
        assert (got[1][~mine] == 7.0).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("news,group,kv_heads,how", [
    ([1], 1, 1, 0), ([1, 1, 1], 4, 2, 1), ([2, 31, 0, 5], 1, 3, 2), ([32, 33], 1, 2, 3), ([63, 64, 65], 2, 1, 0),
    ([200], 3, 2, 1), ([127, 1, 129], 5, 1, 2), ([17], 40, 1, 3), ([300, 128, 77], 2, 2, 0)])
def test_prompts(ctx, io, dim, news, group, kv_heads, how):
    p = Prompts(dim + sum(news), news, [0] * len(news), kv_heads, group, dim, io, how)
    p.check(p.run(ctx))


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("news,priors,group,kv_heads,how", [
    ([1], [1], 2, 1, 0), ([1, 1], [700, 3], 4, 2, 1), ([16, 3, 1], [1000, 0, 4001], 2, 2, 2), ([70, 129], [333, 2000], 2, 1, 3),
    ([8], [9000], 8, 1, 0), ([33, 5, 0], [0, 63, 9], 3, 2, 1)])
def test_after_a_prefix(ctx, io, dim, news, priors, group, kv_heads, how):
    p = Prompts(dim + sum(priors), news, priors, kv_heads, group, dim, io, how)
    p.check(p.run(ctx))


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim,new,prior,heads", [(64, 1, 5000, 1), (96, 20, 3000, 2), (128, 64, 6000, 1), (256, 100, 2500, 1),
                                                 (128, 300, 20000, 1)])
def test_split_keys(ctx, io, dim, new, prior, heads):
    """Few rows over many keys: parts through the workspace, and a launch that joins them."""
    p = Prompts(new, [new, 1], [prior, 0], heads, 2, dim, io)
    batch = p.batch()
    assert ctx.prompt_attention_workspace_bytes(batch, p.q.shape[0], p.k.shape[0], 2 * heads, heads, dim, d._dtype_code(p.q)) > 0
    p.check(p.run(ctx))


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_many_sequences(ctx, io):
    rng = np.random.default_rng(5)
    news = rng.integers(0, 90, 150).tolist()
    p = Prompts(1, news, [0] * 150, 2, 2, 64, io, 1)
    assert ctx.prompt_attention_workspace_bytes(p.batch(), sum(news), sum(news), 4, 2, 64, d._dtype_code(p.q)) == 0
    p.check(p.run(ctx))


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_prompt(ctx, io, dim):
    p = Prompts(3, [2500, 900], [0, 0], 1, 2, dim, io, 1)
    p.check(p.run(ctx))


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("news,nks", [([10, 5], [4, 5]), ([40], [0]), ([100, 7], [30, 0]), ([3], [1])])
def test_fewer_keys_than_rows(ctx, io, news, nks):
    """The first rows see nothing: 0 and -inf."""
    p = Prompts(9, news, [k - n for k, n in zip(nks, news)], 2, 2, 64, io, 0, key_spare=2)
    got = p.run(ctx)
    p.check(got)
    if nks[0] < news[0]:
        assert (got[1][0] == float("-inf")).all() and (got[0][0] == 0).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("prior", [0, 3000])
def test_rows_left_out(ctx, io, prior):
    """Rows behind the last sequence, and past max_new, are left as they were."""
    p = Prompts(11, [50, 20], [prior, 0], 1, 2, 128, io, 0, spare=9, key_spare=3)
    out = torch.full_like(p.q, 5.0)
    p.check(p.run(ctx, out=out))
    assert (out[70:] == 5.0).all()
    out.fill_(5.0)
    got = p.run(ctx, out=out, batch=p.batch(max_new=33))
    p.check(got, most=33)
    assert (out[33:50] == 5.0).all() and (got[1][33:50] == 7.0).all()


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0, 1.5, 1e-4])
@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_scales(ctx, scale, io):
    p = Prompts(13, [90, 7], [0, 40], 2, 2, 64, io, 1)
    p.check(p.run(ctx, scale=scale), scale)


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_large_scores(ctx, io):
    """Scores far apart, and a running maximum that keeps growing: later keys outweigh all before."""
    p = Prompts(15, [260], [0], 1, 1, 64, io)
    ramp = torch.linspace(0.1, 30, 260, device="cuda")[:, None, None]
    p.k, p.q = (p.k.float() * ramp).to(DT[io]), (p.q.float() * 3).to(DT[io])
    p.check(p.run(ctx))
    p.k = (p.k.float().abs() * 2.0**18).to(DT[io])  # scores up to 2^30
    p.q = p.q.abs()
    got = p.run(ctx)
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()
    s = (p.q[:, 0].double() @ p.k[:, 0].double().T.contiguous()) * 0.125
    best = s.masked_fill(~torch.ones_like(s, dtype=torch.bool).tril(), float("-inf")).argmax(-1)
    top2 = s.masked_fill(~torch.ones_like(s, dtype=torch.bool).tril(), float("-inf")).topk(2, -1).values
    clear = top2[:, 0] - top2[:, 1] > 80 * 2.0**-24 * top2[:, 0] * 2 + 40  # beyond the scores' error by e^40
    assert clear.sum() > 50
    want = p.v[best, 0][clear].double()  # one probability, rounded; its quotient by the sum; the output's rounding
    assert ((got[0][clear, 0].double() - want).abs() <= (P_STEP[io] + HALF_STEP[io] + 4 * 2.0**-24) * want.abs()).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("news,priors", [([70, 200, 3], [0, 0, 0]), ([9, 40], [3000, 20])])
def test_masked_values_have_no_influence(ctx, io, dim, news, priors):
    """NaN and infinities in keys and values that a row does not see: the rows before see none of
    them, bit by bit; those that see them become what the sum is."""
    p = Prompts(17, news, priors, 2, 2, dim, io, 1, spare=5, key_spare=5)
    clean = p.run(ctx)
    p.k, p.v = p.k.clone(), p.v.clone()
    p.k[p.key_starts[-1]:], p.v[p.key_starts[-1]:] = float("nan"), float("inf")
    again = p.run(ctx)
    assert torch.equal(clean[0][:sum(news)], again[0][:sum(news)]) and torch.equal(clean[1], again[1])
    b = 1  # one value infinite late in this sequence, the key of another NaN
    row, key_row = news[b] - 2, news[b] - 1
    at = int(p.key_starts[b]) + priors[b]
    p.v[at + row, 0, 5], p.v[at + row, 1, 7] = float("inf"), float("nan")
    p.k[at + key_row, 1, 3] = float("nan")
    got = p.run(ctx)
    out, lse, tol, ltol = p.expect(dim**-0.5)
    r0 = int(p.starts[b])
    before = torch.ones(sum(news), dtype=torch.bool, device="cuda")
    before[r0 + row:r0 + news[b]] = False
    e = ((got[0][:sum(news)].double() - out[:sum(news)]).abs() / tol[:sum(news)])[before]
    assert (e <= 1).all(), e.max()
    assert ((got[1][:sum(news)].double() - lse[:sum(news)]).abs() <= ltol[:sum(news)])[before].all()
    y = got[0].float()
    assert (y[r0 + row, :2, 5] == float("inf")).all() and torch.isnan(y[r0 + row, 2:, 7]).all()
    others = torch.ones(dim, dtype=torch.bool, device="cuda")
    others[5] = others[7] = False
    assert torch.isfinite(y[r0 + row][:, others]).all()
    assert torch.isnan(y[r0 + key_row, 2:]).all() and torch.isnan(got[1][r0 + key_row, 2:]).all()
    assert (y[r0 + key_row, :2, 5] == float("inf")).all() and torch.isfinite(y[r0 + key_row, :2][:, others]).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_strides_beyond_32_bits(ctx, io):
    n, dim, stride = 3, 64, (1 << 30) + 64 if io == "f32" else (1 << 31) + 64
    flat = torch.empty(2 * stride + 8 * dim, dtype=DT[io], device="cuda")
    view = lambda at, h: flat[at * dim:].as_strided((n, h, dim), (stride, dim, 1))
    p = Prompts(19, [n], [0], 1, 2, dim, io)
    q, k, v, out = view(0, 2), view(2, 1), view(3, 1), view(4, 2)
    for a, b in ((q, p.q), (k, p.k), (v, p.v)):
        a.copy_(b)
    p.q, p.k, p.v = q, k, v
    p.check(p.run(ctx, out=out))


def test_output_layouts(ctx):
    for io in ("bf16", "f32"):
        p = Prompts(21, [77, 30], [0, 0], 2, 3, 96, io)
        want = p.run(ctx)[0]
        for how in ("odd", "head_major", "fused"):
            out, _ = rows(p.rng, 107, 6, 96, DT[io], how)
            assert torch.equal(p.run(ctx, out=out)[0], want)


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("prior", [0, 4000])
def test_same_every_time_and_in_a_graph(ctx, io, prior):
    p = Prompts(23, [130, 60], [prior, 0], 2, 2, 128, io)
    first = p.run(ctx)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, p.run(ctx)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ctx.prompt_attention(p.q, p.k, p.v, p.batch(), stream=side)
    side.synchronize()
    assert torch.equal(got, first[0])
    batch, out = p.batch(), torch.empty_like(p.q)
    lse = torch.empty(p.q.shape[:2], device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.prompt_attention(p.q, p.k, p.v, batch, out=out, lse=lse)
    for _ in range(3):
        p.q.copy_(torch.randn_like(p.q))
        g.replay()
        torch.cuda.synchronize()
        want = p.run(ctx)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_nothing_to_do(ctx):
    q = torch.empty(0, 4, 64, device="cuda")
    assert ctx.prompt_attention(q, q, q, d.PromptBatch(i32([0]), 0)).shape == (0, 4, 64)
    q = torch.ones(3, 4, 64, device="cuda")
    out = torch.full_like(q, 2.0)
    ctx.prompt_attention(q, q, q, d.PromptBatch(i32([0, 0, 0]), 0), out=out)  # no sequence has rows
    assert (out == 2.0).all()
    k = torch.empty(0, 2, 64, device="cuda")
    assert (ctx.prompt_attention(q, k, k, d.PromptBatch(i32([0, 3]), 3, i32([0, 0]), 0)) == 0).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("news,priors,told", [([9], [9000], 3000), ([9], [9000], 0), ([200, 3], [700, 2500], 64), ([40], [0], 1)])
def test_more_keys_than_told(ctx, io, news, priors, told):
    """max_keys shapes the launch only: parts grow, and none is lost."""
    for dim in (64, 256):
        p = Prompts(25, news, priors, 1, 4, dim, io)
        p.check(p.run(ctx, batch=d.PromptBatch(i32(p.starts), max(news), i32(p.key_starts), told)))


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_starts_outside(ctx, io):
    """Starts outside the rows count as the nearest; a sequence that ends before it starts has no rows."""
    p = Prompts(27, [60, 40], [0, 0], 1, 2, 64, io)
    p.starts[-1] = p.key_starts[-1] = 100
    want = p.run(ctx)
    p.check(want)
    for starts in ([-7, 60, 100], [0, 60, 2**31 - 1], [-2**31, 60, 101]):
        got = p.run(ctx, batch=d.PromptBatch(i32(starts), 60))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = torch.full_like(p.q, 5.0)
    got = p.run(ctx, out=out, batch=d.PromptBatch(i32([60, 0, 60]), 60))
    assert torch.equal(got[0][:60], want[0][:60]) and (out[60:] == 5.0).all() and (got[1][60:] == 7.0).all()


def test_refused(ctx):
    q, k = torch.ones(6, 4, 64, device="cuda"), torch.ones(9, 2, 64, device="cuda")
    batch = d.PromptBatch(i32([0, 6]), 6, i32([0, 9]), 9)
    good = dict(q=q, k=k, v=k, batch=batch)
    assert torch.equal(ctx.prompt_attention(**good), torch.ones_like(q))
    for bad in (dict(q=q[0]), dict(q=q.cpu()), dict(q=q.transpose(0, 2)), dict(k=k.half()), dict(v=k[:8]), dict(v=k[:, :1]),
                dict(k=k.bfloat16()), dict(k=k[:, :, :32]), dict(batch=d.PromptBatch(i32([0, 6]), 6)),
                dict(batch=d.PromptBatch(i32([0, 6]).long(), 6, i32([0, 9]), 9)), dict(batch=d.PromptBatch(i32([]), 6, i32([]), 9)),
                dict(batch=d.PromptBatch(i32([0, 6]), 7, i32([0, 9]), 9)), dict(batch=d.PromptBatch(i32([0, 6]), -1, i32([0, 9]), 9)),
                dict(batch=d.PromptBatch(i32([0, 6]), 6, i32([0, 9, 9]), 9)), dict(batch=d.PromptBatch(i32([0, 6]), 6, i32([0, 9]), 10)),
                dict(lse=torch.empty(6, 3, device="cuda")), dict(lse=torch.empty(6, 4, device="cuda").double()),
                dict(out=q), dict(out=q.bfloat16()), dict(out=torch.empty(5, 4, 64, device="cuda")), dict(scale=float("nan"))):
        with pytest.raises(d.DyninferError):
            ctx.prompt_attention(**{**good, **bad})
    long = torch.ones(5000, 2, 64, device="cuda")
    with pytest.raises(d.DyninferError):  # parts, and no room for them
        ctx.prompt_attention(q, long, long, d.PromptBatch(i32([0, 6]), 6, i32([0, 5000]), 5000), workspace=torch.empty(256, device="cuda"))


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("news,priors", [([1, 64, 65, 200], [0, 0, 0, 0]), ([33, 9], [2500, 700])])
def test_layouts_have_the_same_bits(ctx, io, dim, news, priors):
    """Rows and outputs on and off 16-byte boundaries, heads apart, and rows between others that stay."""
    p = Prompts(29, news, priors, 2, 3, dim, io)
    want = p.run(ctx)
    p.check(want)
    q, t = p.q, sum(news)
    wide = torch.full((t + 2, 9, dim), 3.0, device="cuda", dtype=DT[io])
    for how in ("odd", "head_major", "fused"):
        out, _ = rows(p.rng, t, 6, dim, DT[io], how)
        p.q, _ = rows(p.rng, t, 6, dim, DT[io], how)
        p.q.copy_(q)
        got = p.run(ctx, out=out)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    p.q = q
    got = p.run(ctx, out=wide[1:-1, 2:8])
    assert torch.equal(got[0], want[0])
    wide[1:-1, 2:8] = 3.0
    assert (wide == 3.0).all()
