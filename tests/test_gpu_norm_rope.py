"""Norms of query and key heads with the rotation, alone and on the way into the cache, on the
GPU through the C ABI, against 64 bits.

Tolerance of a value, in units of 2^-24 of what it is made of: the sum of squares takes 8 + 5
roundings, its mean and eps 3, all halved by the root; v_rsq_f32 2; three products and w + offset 4;
so 14 on a and b, and 2 more in a c - b s: 16 (|a c| + |b s|).  Then half a step of the output's type.
In f32 one pass gives the same bits as its two steps one after the other wherever a lane holds
the same eight dims in both (halves of whole fours hold theirs as pairs, and sum their squares in another order)."""
import numpy as np
import pytest
import torch

import dyninfer_amd as d
import kvref
from test_gpu_kvcache import DT, ENC, HOW, Case, dev, i32, rows

pytestmark = pytest.mark.gpu

HALF_STEP = {"f32": 2.0**-24, "bf16": 2.0**-8}


def normed(x, w, eps, offset):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (w.astype(np.float64) + offset)


def turned(y, table, positions, rot, half):
    """(rotated, sum of the magnitudes of its products) in 64 bits."""
    z, size = y.copy(), np.abs(y)
    if rot == 0:
        return z, size
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    for i, p in enumerate(positions):
        if not 0 <= p < len(table):
            z[i, :, :rot] = np.nan
            continue
        c, s = table[p][:, 0].astype(np.float64), table[p][:, 1].astype(np.float64)
        u, v = y[i][:, a], y[i][:, b]
        z[i][:, a], z[i][:, b] = u * c - v * s, u * s + v * c
        size[i][:, a], size[i][:, b] = np.abs(u * c) + np.abs(v * s), np.abs(u * s) + np.abs(v * c)
    return z, size


def check(got, x, w, eps, offset, table, positions, rot, half, io):
    want, size = turned(normed(x, w, eps, offset), table, positions, rot, half)
    got = got.float().cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    tol = 16 * 2.0**-24 * size + HALF_STEP[io] * np.abs(want) + 1e-44
    assert (np.abs(got - want)[ok] <= tol[ok]).all(), np.max((np.abs(got - want) / tol)[ok])


@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 24), (96, 96), (96, 48), (96, 10), (128, 128), (128, 64), (128, 2),
                                     (256, 256), (256, 96), (128, 0)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv_heads,how", [(1, 1, 1, 0), (1, 16, 8, 1), (37, 5, 5, 2), (130, 7, 3, 3)])
def test_norm_rope(ctx, dim, rot, layout, io, tokens, heads, kv_heads, how):
    rng = np.random.default_rng(dim + rot + tokens)
    q, qf = rows(rng, tokens, heads, dim, DT[io], HOW[how])
    k, kf = rows(rng, tokens, kv_heads, dim, DT[io], HOW[(how + 1) % 4])
    offset, eps = float(how % 2), 10.0 ** -(how + 4)
    wt = [(rng.normal(1 - offset, 0.4, dim)).astype(np.float32) for _ in range(2)]
    types = ["f32", "bf16"] if how % 2 else ["bf16", "f32"]
    wd = [dev(w, DT[t]) for w, t in zip(wt, types)]
    if how == 2:  # a weight off 16-byte boundaries
        wd = [torch.cat([w[:1], w])[1:] for w in wd]
    wt = [w.float().cpu().numpy() for w in wd]
    positions = rng.integers(-1, 41, tokens)  # the first and the last lie outside the table
    table = kvref.table(40, max(rot, 2)).astype(np.float32)
    rope = d.Rope(dev(table), i32(positions), rot, layout) if rot else None
    got_q, got_k = ctx.qk_norm_rope(q, k, rope, q_norm=d.HeadNorm(wd[0], eps, offset), k_norm=d.HeadNorm(wd[1], eps, offset))
    check(got_q, qf, wt[0], np.float32(eps), offset, table, positions, rot, layout == "half", io)
    check(got_k, kf, wt[1], np.float32(eps), offset, table, positions, rot, layout == "half", io)
    assert torch.equal(q.float().cpu(), torch.from_numpy(qf)) and torch.equal(k.float().cpu(), torch.from_numpy(kf))


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dim,rot,layout", [(128, 128, "half"), (128, 64, "half"), (96, 20, "half"), (64, 64, "interleaved"),
                                            (256, 30, "interleaved")])
def test_in_place_and_parts(ctx, io, dim, rot, layout):
    """Into its own rows, slices of one tensor, one of the two alone, a norm on one only: the same values."""
    rng = np.random.default_rng(rot)
    wide = dev(rng.normal(0, 2, (53, 11, dim)).astype(np.float32), DT[io])
    rope = d.Rope(dev(kvref.table(90, rot).astype(np.float32)), i32(rng.integers(0, 90, 53)), rot, layout)
    nq, nk = (d.HeadNorm(dev(rng.normal(1, 0.2, dim).astype(np.float32))) for _ in range(2))
    q, k = wide[:, :7], wide[:, 7:9]
    want_q, want_k = ctx.qk_norm_rope(q.contiguous(), k.contiguous(), rope, nq, nk)
    other = wide[:, 9:].clone()
    assert torch.equal(ctx.qk_norm_rope(q, None, rope, nq)[0], want_q) and ctx.qk_norm_rope(q, None, rope, nq)[1] is None
    a, b = ctx.qk_norm_rope(q, k, rope, nq)  # keys without a norm
    assert torch.equal(a, want_q) and torch.equal(b, ctx.rope(k, rope))
    a, b = ctx.qk_norm_rope(q, k, rope, None, nk)
    assert torch.equal(a, ctx.rope(q, rope)) and torch.equal(b, want_k)
    ones = d.HeadNorm(torch.ones(dim, device="cuda"))
    assert torch.equal(ctx.qk_norm_rope(q, None, rope, d.HeadNorm())[0], ctx.qk_norm_rope(q, None, rope, ones)[0])
    ctx.qk_norm_rope(q, k, rope, nq, nk, q_out=q, k_out=k)
    assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(wide[:, 9:], other)


@pytest.mark.parametrize("dim,rot,layout", [(64, 64, "half"), (96, 48, "half"), (128, 40, "half"), (128, 128, "interleaved"),
                                            (256, 34, "half")])
@pytest.mark.parametrize("kb,vb", [(8, 8), (4, 8), (8, 4), (4, 4)])
def test_same_bits_as_steps(ctx, dim, rot, layout, kb, vb):
    """Norm then rotation, and norm then append, in f32: the bits of the one pass (queries: those of qk_norm_rope)."""
    page, news, lens = (16, [3, 0, 17, 40], [5, 9, 0, 30]) if kb == vb else (64, [1] * 5, [0, 15, 16, 700, 63])
    c = Case(dim + kb + vb, news, lens, 3, dim, page, kb, vb)
    q, _ = rows(c.rng, c.tokens, 6, dim, torch.float32, "fused")
    k, _ = rows(c.rng, c.tokens, 3, dim, torch.bfloat16, "fused")
    v, _ = rows(c.rng, c.tokens, 3, dim, torch.bfloat16, "plain")
    rope = d.Rope(dev(kvref.table(1000, rot).astype(np.float32)), i32(c.rng.integers(0, 1000, c.tokens)), rot, layout)
    nq, nk = (d.HeadNorm(dev(c.rng.normal(0, 0.2, dim).astype(np.float32)), 1e-5, 1.0) for _ in range(2))
    q1, k1 = ctx.qk_norm_rope(q, k.float(), None, nq, nk)
    one_q, one_k = ctx.qk_norm_rope(q, k.float(), rope, nq, nk)
    if layout == "interleaved" or rot % 8:
        assert torch.equal(one_q, ctx.rope(q1, rope)) and torch.equal(one_k, ctx.rope(k1, rope))
    other = d.KVCache(c.cache.k.clone(), c.cache.v.clone(), c.cache.pages, 3, dim, page, ENC[kb], ENC[vb])
    got = ctx.kv_append(c.cache, c.batch, k, v, rope, q=q, q_norm=nq, k_norm=nk)
    ctx.kv_append(other, c.batch, k1, v.float(), rope)
    assert torch.equal(got, one_q)
    assert torch.equal(c.cache.k, other.k) and torch.equal(c.cache.v, other.v)
    # norms without a rotation; a norm of the keys alone; of the queries alone
    got = ctx.kv_append(c.cache, c.batch, k, v, q=q, q_norm=nq, k_norm=nk)
    ctx.kv_append(other, c.batch, k1, v.float())
    assert torch.equal(got, q1) and torch.equal(c.cache.k, other.k)
    assert torch.equal(ctx.kv_append(c.cache, c.batch, k, v, rope, q=q, k_norm=nk), ctx.rope(q, rope))
    ctx.kv_append(other, c.batch, k1, v.float(), rope)
    assert torch.equal(c.cache.k, other.k)
    assert torch.equal(ctx.kv_append(c.cache, c.batch, k, v, rope, q=q, q_norm=nq), one_q)
    ctx.kv_append(other, c.batch, k, v, rope)
    assert torch.equal(c.cache.k, other.k) and torch.equal(c.cache.v, other.v)


def test_magnitudes(ctx):
    """Heads whose squares leave f32, tiny ones, zeros, infinities and NaN; each head by itself."""
    dim = 128
    rng = np.random.default_rng(3)
    x = np.repeat(rng.normal(0, 1, (1, 1, dim)), 12, 1).astype(np.float32)
    scales = [1, 1e19, 3e37, 1e30, 1e-3, 1e-20, 1e-38, 0, 1, 1, 1e25, 1]
    x[0] *= np.array(scales, np.float32)[:, None]
    x[0, 8, 5], x[0, 9, 7] = np.nan, np.inf
    w = rng.normal(1, 0.3, dim).astype(np.float32)
    got = ctx.qk_norm_rope(dev(x), q_norm=d.HeadNorm(dev(w), 1e-6))[0].cpu().numpy().astype(np.float64)
    assert np.isnan(got[0, 8]).all()
    assert np.isnan(got[0, 9, 7]) and (np.delete(got[0, 9], 7) == 0).all()
    fine = [i for i in range(12) if i not in (8, 9)]
    want = normed(x[0, fine], w, np.float32(1e-6), 0)
    assert (np.abs(got[0, fine] - want) <= 16 * 2.0**-24 * np.abs(want) + 1e-44).all()


def test_strides_beyond_32_bits(ctx):
    """Token strides whose offsets pass 2^32 elements."""
    stride, n, dim = (1 << 31) + 64, 3, 64
    flat = torch.empty(2 * stride + 4 * dim, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((n, 2, dim), (stride, dim, 1))
    y = flat[2 * dim:].as_strided((n, 2, dim), (stride, dim, 1))
    x.copy_(torch.randn(n, 2, dim, device="cuda"))
    norm = d.HeadNorm(torch.rand(dim, device="cuda"))
    want = ctx.qk_norm_rope(x.contiguous(), q_norm=norm)[0]
    ctx.qk_norm_rope(x, q_norm=norm, q_out=y)
    assert torch.equal(y, want)


def test_stream_and_graph(ctx):
    x = torch.randn(65, 8, 128, device="cuda", dtype=torch.bfloat16)
    k = torch.randn(65, 2, 128, device="cuda", dtype=torch.bfloat16)
    norm = d.HeadNorm(torch.rand(128, device="cuda"))
    rope = d.Rope(ctx.rope_table(100, 128), i32(np.arange(65)), 128)
    want = ctx.qk_norm_rope(x, k, rope, norm, norm)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ctx.qk_norm_rope(x, k, rope, norm, norm, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    oq, ok = torch.empty_like(x), torch.empty_like(k)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.qk_norm_rope(x, k, rope, norm, norm, q_out=oq, k_out=ok)
    for i in range(3):
        x.copy_(torch.randn(65, 8, 128, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(oq, ctx.qk_norm_rope(x, k, rope, norm, norm)[0])
        assert torch.equal(ok, want[1])


def test_nothing_to_do(ctx):
    x = torch.empty(0, 4, 64, device="cuda")
    out = ctx.qk_norm_rope(x, x, q_norm=d.HeadNorm(), k_norm=d.HeadNorm())
    assert out[0].shape == (0, 4, 64) and out[1].shape == (0, 4, 64)


def test_refused(ctx):
    q, k, w = torch.ones(6, 4, 64, device="cuda"), torch.ones(6, 2, 64, device="cuda"), torch.ones(64, device="cuda")
    rope = d.Rope(ctx.rope_table(16, 64), i32(range(6)), 64)
    good = dict(q=q, k=k, rope=rope, q_norm=d.HeadNorm(w), k_norm=d.HeadNorm(w))
    ctx.qk_norm_rope(**good)
    for bad in (dict(q=q[0]), dict(q=q.cpu(), q_out=q), dict(q=q.half()), dict(k=k[:5]), dict(k=k[:, :, :32]), dict(k=None),
                dict(q_norm=d.HeadNorm(w[:32])), dict(q_norm=d.HeadNorm(w.cpu())), dict(q_norm=d.HeadNorm(w.half())),
                dict(q_norm=d.HeadNorm(torch.ones(128, device="cuda")[::2])), dict(k_norm=d.HeadNorm(w, eps=0.0)),
                dict(k_norm=d.HeadNorm(w, offset=float("inf"))), dict(q_norm=d.HeadNorm(w, eps=1e300)), dict(q_out=q[:, :2]),
                dict(q_out=q[:, :1].expand(6, 4, 64)), dict(k_out=q[:, 1:3]), dict(rope=None, k_norm=None),
                dict(rope=d.Rope(rope.table, rope.positions[:5], 64)), dict(rope=d.Rope(rope.table, rope.positions, 128))):
        with pytest.raises(d.DyninferError):
            ctx.qk_norm_rope(**{**good, **bad})


@pytest.mark.parametrize("dim,rot,layout", [(128, 128, "half"), (96, 64, "interleaved"), (256, 256, "half")])
def test_types_apart(ctx, dim, rot, layout):
    """Queries and keys, and their weights, of different types in one call: as each alone."""
    rng = np.random.default_rng(dim)
    rope = d.Rope(dev(kvref.table(90, rot).astype(np.float32)), i32(rng.integers(0, 90, 29)), rot, layout)
    for a, b, wa, wb in (("f32", "bf16", "f32", "f32"), ("bf16", "f32", "bf16", "f32"), ("bf16", "bf16", "f32", "bf16")):
        q, k = (dev(rng.normal(0, 2, (29, h, dim)).astype(np.float32), DT[t]) for h, t in ((5, a), (2, b)))
        nq, nk = (d.HeadNorm(dev(rng.normal(1, 0.2, dim).astype(np.float32), DT[t])) for t in (wa, wb))
        got = ctx.qk_norm_rope(q, k, rope, nq, nk)
        assert torch.equal(got[0], ctx.qk_norm_rope(q, None, rope, nq)[0]) and torch.equal(got[1], ctx.qk_norm_rope(k, None, rope, nk)[0])


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_magnitudes_of_aligned_rows(ctx, io):
    """Overflowing, tiny, zero, infinite and NaN heads beside ordinary ones: each as alone in rows off 16 bytes."""
    x = torch.randn(9, 4, 128, device="cuda")
    x[1, 0] *= 1e30
    x[1, 1] *= 1e-30
    x[2, 2] = 0
    x[3, 3, 7], x[4, 0, 9], x[5, 1] = float("inf"), float("nan"), 3e38
    x = x.to(DT[io])
    w = torch.rand(128, device="cuda") + 0.5
    rope = d.Rope(ctx.rope_table(20, 128), i32(np.arange(9)), 128)
    off = torch.empty(9 * 4 * 128 + 1, device="cuda", dtype=DT[io])[1:].view(9, 4, 128)
    off.copy_(x)
    got, want = (ctx.qk_norm_rope(t, None, rope, d.HeadNorm(w))[0].float() for t in (x, off))
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert torch.isfinite(got[1]).all() and torch.isfinite(got[5]).all() and (got[2, 2] == 0).all()
