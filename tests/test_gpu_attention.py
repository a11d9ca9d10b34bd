"""Attention over the quantized cache on the GPU, against 64 bits on the same codes.

Bound on an output: with A = sum p |v| and S the largest sum of |q| |k| scale a row sees, a
score is off by at most 2^-24 (d + 16) S (f32 sums in any order and the factors' roundings), and
for f32 queries by 2^-22 of what S would be with every |q| the row's largest (what their two f16
terms leave); p
moves by twice that, by 2^-16 for its two bf16 terms (each leaves half a unit in the last of 8 bits, up
to 2^-8; 2^-23 and less with three), and sums of n terms by 2^-24 n / 4 (four partial sums at
least, each in f32).  A rounding to bf16 adds up to 2^-8 of the output, one to f32 2^-24."""
import numpy as np
import pytest
import torch

import dyninfer_amd as d
import kvref
from test_gpu_kvcache import Case, bad, dev, i32, rows

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def random_tree(rng, n):
    return [-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, n)]


def seen_rows(parents):
    see = np.zeros((len(parents),) * 2, bool)
    for i, p in enumerate(parents):
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
    return see


def words(see, count):
    """Rows of truth values -> int64 words."""
    out = np.zeros((len(see), count), np.uint64)
    for i, r in enumerate(see):
        for j in np.flatnonzero(r):
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def expect(c, qf, sees, scale, f32):
    """(out, lse, bound of out, bound of lse) of all rows; sees: [n, length] of each sequence."""
    out, lse, tol, ltol = [], [], [], []
    dim = c.ref.dim
    for b, (n, l) in enumerate(zip(c.news, c.lens)):
        q = qf[c.starts[b]:c.starts[b] + n].astype(np.float64)
        k, v = (c.ref.rows(c.table[b], 0, l + n, kind) for kind in "kv")
        o, e, mag, dot = kvref.attend(q, k, v, sees[b], scale)
        ds = dot * 2.0 ** -24 * (dim + 16)
        if f32:
            flat = np.broadcast_to(np.abs(q).max(-1, keepdims=True), q.shape)
            ds = ds + kvref.attend(flat, np.abs(k), v, sees[b], scale)[3] * 2.0 ** -22
        rel = 2 * ds + (2.0 ** -23 if f32 else 2.0 ** -16) + 2.0 ** -24 * (32 + (l + n) / 4)
        out.append(o), lse.append(e)
        tol.append(rel[..., None] * mag + (2.0 ** -24 if f32 else 2.0 ** -8) * np.abs(o) + 1e-30)
        ltol.append(ds + 2.0 ** -24 * (32 + (l + n) / 4) + 2.0 ** -22 * (1 + np.abs(np.where(np.isfinite(e), e, 0))))
    return tuple(np.concatenate(x) for x in (out, lse, tol, ltol))


def check(ctx, c, io, q_heads, sees, mask, scale=None, how="plain", **kw):
    q, qf = rows(c.rng, c.tokens, q_heads, c.ref.dim, DT[io], how)
    lse = torch.full((c.tokens, q_heads), float("nan"), device="cuda")
    s = c.ref.dim ** -0.5 if scale is None else scale
    got = ctx.tree_attention(c.cache, c.batch, q, mask=mask, scale=scale, lse=lse, **kw)
    out, want_lse, tol, ltol = expect(c, qf, sees, s, io == "f32")
    err = np.abs(got.float().cpu().numpy().astype(np.float64) - out)
    assert (err <= tol).all(), (err / tol).max()
    got_lse = lse.cpu().numpy().astype(np.float64)
    empty = np.isinf(want_lse)
    assert (got_lse[empty] == -np.inf).all()
    assert (np.abs(got_lse[~empty] - want_lse[~empty]) <= ltol[~empty]).all()
    return got


def chain(news, lens):
    return [np.concatenate([np.ones((n, l), bool), np.tril(np.ones((n, n), bool))], 1) for n, l in zip(news, lens)]


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("kb,vb", [(8, 8), (8, 4), (4, 8), (4, 4)])
def test_types_and_dims(ctx, io, dim, kb, vb):
    news, lens = [1, 5, 3], [0, 77, 300]
    c = Case(dim + kb, news, lens, 2, dim, 32, kb, vb)
    check(ctx, c, io, 6, chain(news, lens), None, how="fused")


@pytest.mark.parametrize("page", [16, 64, 256, 4096])
@pytest.mark.parametrize("news,lens", [
    ([1], [0]), ([1], [1]), ([1], [62]), ([1], [63]), ([1], [64]), ([1], [255]), ([1], [256]), ([1], [1023]),
    ([2, 1, 0, 1], [15, 5000, 9, 16]), ([64], [65]), ([130], [3]), ([33, 65], [500, 1])])
def test_lengths_and_pages(ctx, page, news, lens):
    c = Case(page, news, lens, 1, 64, page, 8, 4, spare=0)
    check(ctx, c, "f32" if page == 16 else "bf16", 3, chain(news, lens), None)


@pytest.mark.parametrize("group,heads", [(1, 5), (2, 1), (3, 2), (7, 1), (8, 2), (16, 1), (17, 1), (40, 1)])
def test_groups(ctx, group, heads):
    news, lens = [1, 4], [90, 33]
    c = Case(group, news, lens, heads, 128, 16, 8, 8)
    check(ctx, c, "bf16", heads * group, chain(news, lens), None, how="odd")


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("news,lens", [([8, 3, 16], [100, 0, 17]), ([64, 64], [0, 130]), ([65, 100, 1], [40, 7, 0]),
                                       ([200], [1000])])
def test_trees(ctx, io, news, lens):
    c = Case(sum(news), news, lens, 2, 64, 16, 8, 8)
    seen = [seen_rows(random_tree(c.rng, n)) for n in news]
    w = -(-max(news) // 64) + (1 if max(news) == 65 else 0)  # a word more than needed, once
    wide = [np.pad(s, ((0, 0), (0, 64 * w - s.shape[1]))) for s in seen]
    for s, n in zip(wide, news):  # bits beyond the sequence's rows mean nothing
        s[:, n:] = c.rng.random(s[:, n:].shape) < 0.5
    mask = dev(np.concatenate([words(s, w) for s in wide]))
    sees = [np.concatenate([np.ones((n, l), bool), s], 1) for s, n, l in zip(seen, news, lens)]
    check(ctx, c, io, 4, sees, mask)


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_rows_that_see_nothing(ctx, io):
    news, lens = [6, 6], [0, 10]
    c = Case(9, news, lens, 2, 64, 16, 8, 8)
    seen = [np.eye(6, dtype=bool) for _ in news]
    seen[0][2] = seen[1][2] = False
    sees = [np.concatenate([np.ones((6, l), bool), s], 1) for s, l in zip(seen, lens)]
    got = check(ctx, c, io, 4, sees, dev(np.concatenate([words(s, 1) for s in seen])))
    assert (got[2] == 0).all() and not (got[8] == 0).all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[0, 40], [700, 260]])
def test_what_is_masked_has_no_influence(ctx, io, lens):
    """NaN and huge scales in rejected siblings, behind the end and on absent pages change no bit."""
    news = [5, 9]
    c = Case(12, news, lens, 2, 64, 16, 8, 8, spare=3)
    seen = [seen_rows(random_tree(c.rng, n)) for n in news]
    for s in seen:
        s[:, 2], s[2, 2] = False, False  # nobody sees row 2, itself included
    mask = dev(np.concatenate([words(s, 1) for s in seen]))
    sees = [np.concatenate([np.ones((n, l), bool), s], 1) for s, n, l in zip(seen, news, lens)]
    state = c.rng.bit_generator.state
    first = check(ctx, c, io, 6, sees, mask)
    for fill in (np.nan, 3e38):
        for b, (n, l) in enumerate(zip(news, lens)):
            for pos in [l + 2] + list(range(l + n, -(-(l + n) // 16) * 16)):
                p = c.table[b][pos // 16]
                c.ref.ks[p, :, pos % 16], c.ref.vs[p, :, pos % 16] = kvref.bf16(np.float32(fill)), kvref.bf16(np.float32(fill))
        used = {int(p) for row in c.table for p in row if p >= 0}
        for p in set(range(c.ref.pages)) - used:
            c.ref.ks[p], c.ref.vs[p] = np.nan, np.nan
        kb, vb = c.ref.buffers()
        c.cache.k.copy_(dev(kb)), c.cache.v.copy_(dev(vb))
        c.rng.bit_generator.state = state
        q, _ = rows(c.rng, c.tokens, 6, 64, DT[io], "plain")
        again = ctx.tree_attention(c.cache, c.batch, q, mask=mask)
        assert torch.equal(again, first)


def test_nan_reaches_only_the_rows_that_see_it(ctx):
    news, lens = [4], [70]
    for kind in ("ks", "vs"):
        c = Case(13, news, lens, 1, 64, 16, 8, 8)
        p = c.table[0][72 // 16]
        getattr(c.ref, kind)[p, :, 72 % 16] = np.nan  # row 2
        c.cache.k.copy_(dev(c.ref.buffers()[0])), c.cache.v.copy_(dev(c.ref.buffers()[1]))
        q, _ = rows(c.rng, 4, 2, 64, torch.float32, "plain")
        out = ctx.tree_attention(c.cache, c.batch, q).cpu()
        assert torch.isfinite(out[:2]).all() and torch.isnan(out[2:]).all()


@pytest.mark.parametrize("lens", [[100], [3000]])
def test_absent_pages_are_not_seen(ctx, lens):
    c = Case(14, [4], lens, 2, 64, 16, 8, 8)
    sees = chain([4], lens)
    for at, to in ((1, -1), (4, c.ref.pages), (5, 1 << 30)):
        c.table[0, at] = to
        sees[0][:, 16 * at:16 * at + 16] = False
    c.batch = c.kv_batch(c.news)
    ref_rows = c.ref.rows
    c.ref.rows = lambda *a: np.nan_to_num(ref_rows(*a))
    check(ctx, c, "f32", 4, sees, None)


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_scales_of_values_and_queries(ctx, io):
    """Values and queries of very different size in one call, scores far apart."""
    news, lens = [3], [500]
    c = Case(15, news, lens, 2, 64, 32, 8, 8)
    c.ref.vs[...] = kvref.bf16(np.exp(c.rng.uniform(-60, 60, c.ref.vs.shape)))
    c.ref.ks[...] = kvref.bf16(np.exp(c.rng.uniform(-9, -4, c.ref.ks.shape)))
    c.cache.k.copy_(dev(c.ref.buffers()[0])), c.cache.v.copy_(dev(c.ref.buffers()[1]))
    check(ctx, c, io, 4, chain(news, lens), None)
    for scale in (0.0, -0.3, 40.0):
        check(ctx, c, io, 4, chain(news, lens), None, scale=scale)


def test_a_wrong_longest_length_costs_only_time(ctx):
    news, lens = [2, 3], [3000, 40]
    c = Case(16, news, lens, 1, 64, 64, 8, 8)
    for told in (0, 5, 100000):
        c.batch.max_length = told
        check(ctx, c, "bf16", 4, chain(news, lens), None)


def test_rows_past_the_tables(ctx):
    """Starts beyond the rows, more rows than max_new: only what is left is written."""
    c = Case(17, [6, 6], [20, 30], 1, 64, 16, 8, 8)
    q, qf = rows(c.rng, 12, 2, 64, torch.float32, "plain")
    out = torch.full_like(q, 7.0)
    batch = d.KVBatch(c.batch.page_table, c.batch.lengths, i32([0, 6, 99]), 12, 4, 40)
    ctx.tree_attention(c.cache, batch, q, out=out)
    c.news, c.tokens = [4, 4], 8
    want, _, tol, _ = expect(c, qf, chain([4, 4], [20, 30]), 0.125, True)
    got = out.cpu().numpy()
    assert (np.abs(got[[0, 1, 2, 3, 6, 7, 8, 9]] - want) <= tol).all()
    assert (got[[4, 5, 10, 11]] == 7).all()


def test_strided_out_stream_workspace_and_graph(ctx):
    news, lens = [3, 7], [2000, 300]
    c = Case(18, news, lens, 2, 128, 64, 8, 4)
    q, _ = rows(c.rng, c.tokens, 8, 128, torch.bfloat16, "fused")
    a = ctx.tree_attention(c.cache, c.batch, q)
    for how in ("fused", "odd", "head_major"):
        out, _ = rows(c.rng, c.tokens, 8, 128, torch.bfloat16, how)
        ctx.tree_attention(c.cache, c.batch, q, out=out)
        assert torch.equal(out, a)
    need = ctx.tree_attention_workspace_bytes(c.cache, c.batch, 8, d.DTYPE_BF16)
    assert need > 0
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b = ctx.tree_attention(c.cache, c.batch, q, stream=s, workspace=work)
    e = ctx.tree_attention(c.cache, c.batch, q, stream=s)
    s.synchronize()
    assert torch.equal(a, b) and torch.equal(a, e)
    g, out = torch.cuda.CUDAGraph(), torch.empty_like(a)
    with torch.cuda.graph(g):
        ctx.tree_attention(c.cache, c.batch, q, out=out, workspace=work)
    for _ in range(3):
        out.zero_(), work.fill_(255)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, a)


def test_offsets_beyond_32_bits(ctx):
    """A cache of more than 4 GiB: the last pages' rows, written, read and attended to."""
    pages, page, heads, dim = 3000, 4096, 3, 128
    cache = d.KVCache.empty(pages, heads, dim, page)
    assert cache.k.numel() > 1 << 32
    n = 300
    table = i32([[pages - 1]])
    batch = d.KVBatch(table, i32([0]), i32([0, n]), n, n, n)
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v, q = (torch.randn((n, heads, dim), device="cuda", generator=gen) for _ in range(3))
    ctx.kv_append(cache, batch, k, v)
    near = d.KVCache.empty(2, heads, dim, page)
    first = d.KVBatch(i32([[1]]), i32([0]), i32([0, n]), n, n, n)
    ctx.kv_append(near, first, k, v)
    for a, b in zip(ctx.kv_read(cache, batch), ctx.kv_read(near, first)):
        assert torch.equal(a, b)
    assert torch.equal(ctx.tree_attention(cache, batch, q), ctx.tree_attention(near, first, q))


def test_refusals(ctx):
    c = Case(2, [4], [10], 2, 64, 16, 8, 8)
    q = torch.zeros((4, 4, 64), device="cuda")
    run = lambda q=q, **kw: ctx.tree_attention(c.cache, c.batch, q, **kw)
    bad(lambda: run(q=q.cpu()))
    bad(lambda: run(q=q[:, :3]))                             # not a multiple of the kv heads
    bad(lambda: run(q=q[:3]))
    bad(lambda: run(q=q.half()), d.ERR_UNSUPPORTED)
    bad(lambda: run(out=q.bfloat16()))
    bad(lambda: run(out=q))                                  # in place
    bad(lambda: run(out=torch.zeros((1, 4, 64), device="cuda").expand(4, 4, 64)))
    bad(lambda: run(mask=torch.zeros((4, 0), dtype=torch.int64, device="cuda")))
    bad(lambda: run(mask=torch.zeros((3, 1), dtype=torch.int64, device="cuda")))
    bad(lambda: run(mask=torch.zeros((4, 1), dtype=torch.int32, device="cuda")))
    bad(lambda: run(lse=torch.zeros((4, 2), device="cuda")))
    bad(lambda: run(scale=float("nan")))
    c = Case(2, [4], [3000], 2, 64, 16, 8, 8)
    bad(lambda: ctx.tree_attention(c.cache, c.batch, q, workspace=torch.empty(16, dtype=torch.uint8, device="cuda")))
    need = ctx.tree_attention_workspace_bytes(c.cache, c.batch, 4)
    bad(lambda: ctx.tree_attention(c.cache, c.batch, q, workspace=torch.empty(need + 256, dtype=torch.uint8, device="cuda")[16:]))
    bad(lambda: ctx.tree_attention_workspace_bytes(c.cache, c.batch, 3))


@pytest.mark.parametrize("count", [64, 65, 200])
def test_many_sequences(ctx, count):
    """Some without new tokens, one long: shares begin in the middle of the sequences."""
    rng = np.random.default_rng(count)
    news, lens = rng.integers(0, 3, count).tolist(), rng.integers(0, 90, count).tolist()
    news[count - 2], lens[count - 2] = 2, 2500
    c = Case(18, news, lens, 1, 64, 16, 8, 4)
    check(ctx, c, "bf16", 2, chain(news, lens), None)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("count,news,lens", [(130, (33, 65), 50), (300, (0, 3), 600)])
def test_many_units(ctx, io, count, news, lens):
    """Units of 33 to 64 rows, and units of few steps, in calls with very many of them."""
    rng = np.random.default_rng(count)
    news, lens = rng.integers(*news, count).tolist(), rng.integers(0, lens, count).tolist()
    c = Case(19, news, lens, 1, 64, 16, 8, 8)
    check(ctx, c, io, 1, chain(news, lens), None)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("heads,group,news,lens", [
    (16, 1, [300] * 15 + [1, 257], [0] * 10 + [33] * 7),  # units of many row tiles, whole
    (4, 4, [700, 130], [0, 500]), (8, 3, [1500, 0, 64], [0, 9, 2000])])
def test_prompts(ctx, io, heads, group, news, lens):
    """Long chains: a row tile stops at its last row's own position."""
    c = Case(20, news, lens, heads, 64, 64, 8, 8)
    check(ctx, c, io, heads * group, chain(news, lens), None)


def test_a_prompt_in_whole_units(ctx):
    """Row tiles many and long enough that they are not cut: the first and last rows of some."""
    n, heads = 4500, 8
    c = Case(21, [n], [0], heads, 64, 256, 8, 8)
    assert ctx.tree_attention_workspace_bytes(c.cache, c.batch, heads, d.DTYPE_BF16) > 0
    q, qf = rows(c.rng, n, heads, 64, torch.bfloat16, "plain")
    got = ctx.tree_attention(c.cache, c.batch, q).float().cpu().numpy()
    k, v = (c.ref.rows(c.table[0], 0, n, kind) for kind in "kv")
    for i in (0, 1, 63, 64, 255, 256, 257, 1023, 1024, 2049, 4351, 4352, n - 1):
        o, _, mag, dot = kvref.attend(qf[i:i + 1].astype(np.float64), k[:i + 1], v[:i + 1], np.ones((1, i + 1), bool), 0.125)
        rel = 2 * dot * 2.0 ** -24 * (64 + 16) + 2.0 ** -16 + 2.0 ** -24 * (32 + n / 4)
        assert (np.abs(got[i] - o[0]) <= rel[0][:, None] * mag[0] + 2.0 ** -8 * np.abs(o[0]) + 1e-30).all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("kb,vb", [(8, 8), (8, 4), (4, 8), (4, 4)])
@pytest.mark.parametrize("group,news,lens,told", [
    (4, [6, 5, 8], [300, 0, 700], 200000), (6, [5, 0, 3], [90, 7, 400], 300000),
    (4, [40, 33, 1], [200, 0, 513], 200000), (5, [70, 9, 64], [0, 300, 150], 100000)])
def test_tiles_of_long_calls(ctx, io, dim, kb, vb, group, news, lens, told):
    """The row tiles that calls of much work take, on small data by a longest length that is told."""
    c = Case(dim + kb + vb, news, lens, 2, dim, 32, kb, vb)
    c.batch.max_length = told
    trees = [seen_rows(random_tree(c.rng, n))[:n, :n] for n in news]
    sees = [np.concatenate([np.ones((n, l), bool), t], 1) for n, l, t in zip(news, lens, trees)]
    check(ctx, c, io, 2 * group, sees, dev(np.concatenate([words(t, 2) for t in trees])))
