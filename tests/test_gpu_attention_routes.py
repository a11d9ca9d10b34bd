"""Every kernel that attention's plan can choose, against 64 bits on the same codes; the bounds are
those of test_gpu_attention.  Which tiles a call takes is pinned by its workspace: parts of
(units + shares) tiles of 16 t rows, each row's dims and two statistics in f32, and two numbers a
unit; a call of whole units takes an empty one."""
import numpy as np
import pytest
import torch

import dyninfer_amd as d
import kvref
from test_gpu_attention import DT, chain, check, expect, random_tree, seen_rows, words
from test_gpu_kvcache import Case, dev, i32, rows

pytestmark = pytest.mark.gpu

STEP = 128  # positions of a step


def parts_bytes(seqs, heads, dim, rows_of_head, told, tiles):
    """The workspace of a call in shares whose row tiles are `tiles` times 16 rows."""
    units = seqs * heads * -(-rows_of_head // (16 * tiles))
    shares = min(units * (-(-told // STEP) + 2), 256 if dim > 128 or tiles == 16 else 512)
    return (units + shares) * 16 * tiles * (4 * dim + 8) + 8 * units


def tree_masks(c, count):
    """(sees, mask) of a random tree for each sequence."""
    trees = [seen_rows(random_tree(c.rng, n)) for n in c.news]
    sees = [np.concatenate([np.ones((n, l), bool), t], 1) for n, l, t in zip(c.news, c.lens, trees)]
    return sees, dev(np.concatenate([words(t, count) for t in trees]))


ROUTES = [  # dims, type, group, new rows, lengths, told longest length, tiles
    ((64, 96, 128, 256), "bf16", 2, [3, 5, 1], [300, 0, 700], 3000, 1),
    ((64, 96, 128, 256), "f32", 2, [3, 5, 1], [300, 0, 700], 3000, 1),
    ((64, 96, 128), "f32", 4, [6, 5, 8], [300, 0, 700], 2500, 1),   # two row tiles of 16, as are the next
    ((256,), "bf16", 4, [6, 5, 8], [300, 0, 700], 200000, 1),
    ((256,), "f32", 4, [6, 5, 8], [300, 0, 700], 200000, 1),
    ((64, 96, 128), "bf16", 4, [12, 9, 1], [300, 0, 513], 200000, 2),
    ((64, 96, 128), "bf16", 4, [12, 9, 1], [300, 0, 513], 2500, 4),
    ((64, 96, 128, 256), "f32", 4, [12, 9, 1], [300, 0, 513], 200000, 4),
    ((256,), "bf16", 4, [40, 33, 1], [200, 0, 513], 200000, 4),
    ((256,), "f32", 5, [70, 9, 64], [0, 300, 150], 100000, 4),
    ((64, 96, 128), "bf16", 5, [20, 9, 25], [200, 0, 513], 200000, 8),
    ((96, 128), "bf16", 5, [40, 33, 1], [200, 0, 513], 200000, 16),
    ((96, 128), "f32", 5, [40, 33, 1], [200, 0, 513], 200000, 16),
]


@pytest.mark.parametrize("dim,io,group,news,lens,told,tiles",
                         [(dim, *r[1:]) for r in ROUTES for dim in r[0]])
@pytest.mark.parametrize("kb,vb", [(8, 8), (8, 4), (4, 8), (4, 4)])
def test_shares(ctx, kb, vb, dim, io, group, news, lens, told, tiles):
    """Trees and chains through every row tile, with the launch that joins the parts."""
    c = Case(tiles + dim + kb + vb, news, lens, 2, dim, 32, kb, vb)
    c.batch.max_length = told
    need = ctx.tree_attention_workspace_bytes(c.cache, c.batch, 2 * group, d.DTYPE_F32 if io == "f32" else d.DTYPE_BF16)
    assert need == parts_bytes(len(news), 2, dim, max(news) * group, told, tiles)
    sees, mask = tree_masks(c, 2)
    check(ctx, c, io, 2 * group, sees, mask, how="fused")
    check(ctx, c, io, 2 * group, chain(news, lens), None)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("kb,vb", [(8, 8), (8, 4), (4, 8), (4, 4)])
def test_whole_units_of_many_rows(ctx, io, dim, kb, vb):
    """Row tiles of 64, a workgroup each: no parts, so an empty workspace is enough."""
    news, lens = [12, 40, 1], [20, 0, 90]
    c = Case(dim + kb + vb, news, lens, 2, dim, 16, kb, vb)
    sees, mask = tree_masks(c, 1)
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    check(ctx, c, io, 8, sees, mask, workspace=none)
    check(ctx, c, io, 8, chain(news, lens), None, workspace=none)


@pytest.mark.parametrize("dim,kb,vb,io,heads,n", [
    (64, 8, 8, "bf16", 32, 4500), (96, 8, 4, "bf16", 32, 4200),  # row tiles of 128
    (128, 4, 8, "bf16", 16, 1500), (128, 8, 8, "f32", 16, 4200),  # of 64
    (256, 8, 8, "bf16", 32, 1100), (256, 4, 4, "f32", 32, 1100)])
def test_prompts_in_whole_units(ctx, dim, kb, vb, io, heads, n):
    """Prompts whose row tiles are a workgroup each, the longest first: the first and last rows of some."""
    c = Case(dim + n, [n], [0], heads, dim, 256, kb, vb)
    q, qf = rows(c.rng, n, heads, dim, DT[io], "plain")
    lse = torch.full((n, heads), float("nan"), device="cuda")
    got = ctx.tree_attention(c.cache, c.batch, q, lse=lse, workspace=torch.empty(0, dtype=torch.uint8, device="cuda"))
    got, lse = got.float().cpu().numpy(), lse.cpu().numpy().astype(np.float64)
    k, v = (c.ref.rows(c.table[0], 0, n, kind) for kind in "kv")
    f32 = io == "f32"
    for i in sorted({0, 1, 31, 32, 63, 64, 127, 128, 129, 255, 256, 1023, 1024, n // 64 * 64 - 1, n // 64 * 64, n - 1}):
        qi = qf[i:i + 1].astype(np.float64)
        sees = np.ones((1, i + 1), bool)
        o, e, mag, dot = kvref.attend(qi, k[:i + 1], v[:i + 1], sees, dim ** -0.5)
        ds = dot * 2.0 ** -24 * (dim + 16)
        if f32:
            flat = np.broadcast_to(np.abs(qi).max(-1, keepdims=True), qi.shape)
            ds = ds + kvref.attend(flat, np.abs(k[:i + 1]), v[:i + 1], sees, dim ** -0.5)[3] * 2.0 ** -22
        sums = 2.0 ** -24 * (32 + (i + 1) / 4)
        rel = 2 * ds + (2.0 ** -23 if f32 else 2.0 ** -16) + sums
        tol = rel[0][:, None] * mag[0] + (2.0 ** -24 if f32 else 2.0 ** -8) * np.abs(o[0]) + 1e-30
        assert (np.abs(got[i] - o[0]) <= tol).all(), i
        assert (np.abs(lse[i] - e[0]) <= ds[0] + sums + 2.0 ** -22 * (1 + np.abs(e[0]))).all(), i


MANY = [("bf16", None), ("bf16", 200000), ("f32", None), ("f32", 200000)]  # row tiles of 64, 256, 64, 256


def many(seed, told, dim=128):
    """160 and 100 rows a head over pages of 16 positions."""
    c = Case(seed, [25, 40], [700, 40], 2, dim, 16, 8, 8, spare=3)
    if told:
        c.batch.max_length = told
    return c


@pytest.mark.parametrize("io,told", MANY)
def test_many_rows_that_see_nothing(ctx, io, told):
    c = many(40, told)
    c.lens[1] = 0
    c.batch.lengths = i32(c.lens)
    seen = [seen_rows(random_tree(c.rng, n)) for n in c.news]
    for s in seen:
        s[::3] = False
    sees = [np.concatenate([np.ones((n, l), bool), s], 1) for s, n, l in zip(seen, c.news, c.lens)]
    got = check(ctx, c, io, 8, sees, dev(np.concatenate([words(s, 1) for s in seen])))
    assert (got[25::3] == 0).all() and not (got[:25] == 0).all(-1).any()


@pytest.mark.parametrize("io,told", MANY)
def test_masked_contents_of_many_rows(ctx, io, told):
    """NaN and huge scales in rejected siblings, behind the end and on unused pages change no bit."""
    c = many(41, told)
    seen = [seen_rows(random_tree(c.rng, n)) for n in c.news]
    for s in seen:
        s[:, 2], s[2, 2] = False, False
    mask = dev(np.concatenate([words(s, 1) for s in seen]))
    sees = [np.concatenate([np.ones((n, l), bool), s], 1) for s, n, l in zip(seen, c.news, c.lens)]
    state = c.rng.bit_generator.state
    first = check(ctx, c, io, 8, sees, mask)
    for fill in (np.nan, 3e38):
        for b, (n, l) in enumerate(zip(c.news, c.lens)):
            for pos in [l + 2] + list(range(l + n, -(-(l + n) // 16) * 16)):
                p = c.table[b][pos // 16]
                c.ref.ks[p, :, pos % 16] = c.ref.vs[p, :, pos % 16] = kvref.bf16(np.float32(fill))
        used = {int(p) for row in c.table for p in row if p >= 0}
        for p in set(range(c.ref.pages)) - used:
            c.ref.ks[p], c.ref.vs[p] = np.nan, np.nan
        kb, vb = c.ref.buffers()
        c.cache.k.copy_(dev(kb)), c.cache.v.copy_(dev(vb))
        c.rng.bit_generator.state = state
        q, _ = rows(c.rng, c.tokens, 8, 128, DT[io], "plain")
        assert torch.equal(ctx.tree_attention(c.cache, c.batch, q, mask=mask), first)


@pytest.mark.parametrize("io,told", MANY)
@pytest.mark.parametrize("kind", ["ks", "vs"])
def test_nan_reaches_only_the_rows_of_many_that_see_it(ctx, io, told, kind):
    c = many(42, told)
    pos = 40 + 17  # row 17 of the second sequence
    getattr(c.ref, kind)[c.table[1][pos // 16], :, pos % 16] = np.nan
    kb, vb = c.ref.buffers()
    c.cache.k.copy_(dev(kb)), c.cache.v.copy_(dev(vb))
    q, _ = rows(c.rng, c.tokens, 8, 128, DT[io], "plain")
    lse = torch.zeros((c.tokens, 8), device="cuda")
    out = ctx.tree_attention(c.cache, c.batch, q, lse=lse)
    assert torch.isfinite(out[:25 + 17]).all() and torch.isnan(out[25 + 17:]).all()
    assert torch.isfinite(lse[:25 + 17]).all() and torch.isnan(lse[25 + 17:]).all() == (kind == "ks")


@pytest.mark.parametrize("io,told", MANY)
def test_absent_pages_of_many_rows(ctx, io, told):
    c = many(43, told)
    sees = chain(c.news, c.lens)
    for at, to in ((0, -1), (3, c.ref.pages), (14, 1 << 30), (44, -5)):  # the last holds rows of the call
        c.table[0, at] = to
        sees[0][:, 16 * at:16 * at + 16] = False
    c.batch = c.kv_batch(c.news)
    if told:
        c.batch.max_length = told
    ref_rows = c.ref.rows
    c.ref.rows = lambda *a: np.nan_to_num(ref_rows(*a))
    check(ctx, c, io, 8, sees, None)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("how", ["fused", "odd", "head_major"])
@pytest.mark.parametrize("news,lens", [([3, 7], [2000, 30]), ([3, 7], [90, 30]), ([30, 17], [700, 30]), ([30, 17], [60, 30])])
def test_strided_outputs(ctx, io, how, news, lens):
    """Outputs of other strides, in shares and whole units, of few rows and many."""
    c = Case(44, news, lens, 2, 128, 64, 8, 4)
    out, _ = rows(c.rng, c.tokens, 8, 128, DT[io], how)
    got = check(ctx, c, io, 8, chain(news, lens), None, how=how, out=out)
    assert got.data_ptr() == out.data_ptr()


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_strides_beyond_32_bits(ctx, io):
    """Tokens more than 2^31 elements apart, in everything a step of one layer reads and writes."""
    c = Case(45, [2, 1], [30, 7], 2, 64, 16, 8, 8)
    n, rot, gap = 3, 64, (1 << 31) + 64
    base = torch.empty((n - 1) * gap + 64 * 64, dtype=DT[io], device="cuda")
    far = lambda first, heads: base.as_strided((n, heads, rot), (gap, rot, 1), 64 * first)
    q, k, v, qr, out, k2, v2 = (far(f, h) for f, h in ((0, 4), (4, 2), (6, 2), (8, 4), (12, 4), (16, 2), (18, 2)))
    near = [rows(c.rng, n, h, rot, DT[io], "plain") for h in (4, 2, 2)]
    for to, (x, _) in zip((q, k, v), near):
        to.copy_(x)
    table = ctx.rope_table(64, rot)
    pos = i32([30, 31, 7])
    rope = d.Rope(table, pos, rot)
    ctx.kv_append(c.cache, c.batch, k, v, rope=rope, q=q, q_out=qr)
    turned = [kvref.rotate(x, table.cpu().numpy(), pos.tolist(), rot, True) for _, x in near[:2]]
    c.write(turned[1], near[2][1])
    assert c.same_bytes()
    as_io = lambda x: dev(x.astype(np.float32), DT[io])
    assert torch.equal(qr.contiguous(), as_io(turned[0]))
    ctx.rope(q, rope, out=out)
    assert torch.equal(out.contiguous(), as_io(turned[0]))
    ctx.kv_read(c.cache, c.batch, k_out=k2, v_out=v2)
    want = [np.concatenate([c.ref.rows(c.table[b], l, m, kind) for b, (m, l) in enumerate(zip(c.news, c.lens))]) for kind in "kv"]
    assert torch.equal(k2.contiguous(), as_io(want[0])) and torch.equal(v2.contiguous(), as_io(want[1]))
    ctx.tree_attention(c.cache, c.batch, qr, out=out)
    o, _, tol, _ = expect(c, qr.float().cpu().numpy(), chain(c.news, c.lens), rot ** -0.5, io == "f32")
    assert (np.abs(out.float().cpu().numpy().astype(np.float64) - o) <= tol).all()


def test_pages_beyond_32_bits(ctx):
    """The last page of a cache of more than 4 GiB, against 64 bits on the codes that were written."""
    pages, page, heads, dim, n = 3000, 4096, 3, 128, 120
    cache = d.KVCache.empty(pages, heads, dim, page)
    assert cache.k.numel() > 1 << 32 and cache.v.numel() > 1 << 32
    batch = d.KVBatch(i32([[pages - 1]]), i32([0]), i32([0, n]), n, n, n)
    rng = np.random.default_rng(46)
    k, v, q = (rng.normal(0, 1, (n, h, dim)).astype(np.float32) for h in (heads, heads, 2 * heads))
    ctx.kv_append(cache, batch, dev(k), dev(v))
    (kc, ks), (vc, vs) = kvref.quant(k, 8, 32), kvref.quant(v, 8, dim)
    k64, v64 = kc * np.repeat(ks.astype(np.float64), 32, -1), vc * vs.astype(np.float64)
    for got, want in zip(ctx.kv_read(cache, batch), (k64, v64)):
        assert np.array_equal(got.cpu().numpy(), want)
    sees = np.tril(np.ones((n, n), bool))
    o, _, mag, dot = kvref.attend(q.astype(np.float64), k64, v64, sees, dim ** -0.5)
    flat = np.broadcast_to(np.abs(q.astype(np.float64)).max(-1, keepdims=True), q.shape)
    ds = dot * 2.0 ** -24 * (dim + 16) + kvref.attend(flat, np.abs(k64), v64, sees, dim ** -0.5)[3] * 2.0 ** -22
    tol = (2 * ds + 2.0 ** -23 + 2.0 ** -24 * (32 + n / 4))[..., None] * mag + 2.0 ** -24 * np.abs(o) + 1e-30
    assert (np.abs(ctx.tree_attention(cache, batch, dev(q)).cpu().numpy() - o) <= tol).all()


@pytest.mark.parametrize("io,news,told", [("bf16", 2, None), ("f32", 2, None), ("bf16", 2, 3000), ("f32", 2, 3000),
                                          ("bf16", 40, None), ("f32", 40, None), ("bf16", 40, 200000), ("f32", 40, 200000)])
def test_scores_beyond_the_exponentials_range(ctx, io, news, told):
    """One key that every row's queries agree with, the others 0: each row gets that key's value, or,
    from scores of 2^30 on, NaN; never 0 as if it saw nothing.  The weights are exactly 1 and 0, so
    that the value is rounded to its terms and to the output's type only."""
    c = Case(47, [news], [700], 1, 64, 16, 8, 8)
    if told:
        c.batch.max_length = told
    c.ref.kc[...] = 0
    p, slot = c.table[0][333 // 16], 333 % 16
    c.ref.kc[p, 0, slot], c.ref.ks[p, 0, slot] = 127, 1
    c.ref.vc[p, 0, slot] = 1 + c.rng.integers(0, 127, 64)
    kb, vb = c.ref.buffers()
    c.cache.k.copy_(dev(kb)), c.cache.v.copy_(dev(vb))
    q = c.rng.uniform(0.5, 1, (news, 4, 64)) * np.exp2(c.rng.uniform(6, 60, (news, 4, 1)))
    q = dev(q.astype(np.float32), DT[io])
    lse = torch.zeros((news, 4), device="cuda")
    got = ctx.tree_attention(c.cache, c.batch, q, lse=lse).double().cpu().numpy()
    score = q.double().sum(-1).cpu().numpy() * 127 / 8
    assert (score < 2.0 ** 29).any() and (score > 2.0 ** 33).any()
    v = c.ref.row(p, slot, "v")[0]
    right = (np.abs(got - v) <= np.abs(v) * (2.0 ** -22 if io == "f32" else 2.0 ** -8 + 2.0 ** -16)).all(-1)
    lost = np.isnan(got).all(-1)
    assert (right | lost).all() and not lost[score < 2.0 ** 30].any()
    lse = lse.cpu().numpy().astype(np.float64)
    assert (np.isnan(lse) == lost).all() and (np.abs(lse - score) <= score * 2.0 ** -16)[right].all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kb", [8, 4])
@pytest.mark.parametrize("news,power", [(2, 97), (40, 97), (2, -110), (40, -110)])
def test_keys_and_queries_far_from_one(ctx, io, kb, news, power):
    """Keys' scales near 2^98, up to where sums of scaled codes stay finite, and very small ones, with
    queries that bring the scores back to ordinary sizes."""
    c = Case(48, [news], [300], 1, 64, 16, kb, 8)
    c.ref.ks[...] = kvref.bf16(c.rng.uniform(0.5, 1, c.ref.ks.shape) * 2.0 ** power)
    kbuf, vbuf = c.ref.buffers()
    c.cache.k.copy_(dev(kbuf)), c.cache.v.copy_(dev(vbuf))
    q = dev((c.rng.normal(0, 1, (news, 4, 64)) * 2.0 ** -(power + 3)).astype(np.float32), DT[io])
    lse = torch.zeros((news, 4), device="cuda")
    got = ctx.tree_attention(c.cache, c.batch, q, lse=lse).double().cpu().numpy()
    out, want, tol, ltol = expect(c, q.float().cpu().numpy(), chain([news], [300]), 0.125, io == "f32")
    assert (np.abs(got - out) <= tol).all() and (np.abs(lse.cpu().numpy() - want) <= ltol).all()
