"""Rotary positions and the quantized paged cache on the GPU, through the C ABI.

Codes, scales, rotations and read-back values are bit-exact with the same f32 operations in
numpy; the rotary table is within one f32 rounding of 64 bits; writes touch no byte that is
not theirs; what lies outside the tables is dropped or reads as NaN."""
import numpy as np
import pytest
import torch

import dyninfer_amd as d
import kvref

pytestmark = pytest.mark.gpu

ENC = {8: d.KV_Q8, 4: d.KV_Q4}
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


class Case:
    """A cache of random contents, sequences on shuffled pages, and their new rows."""

    def __init__(self, seed, news, lens, heads, dim, page, kb, vb, spare=2):
        rng = self.rng = np.random.default_rng(seed)
        need = [max(1, -(-(n + l) // page)) for n, l in zip(news, lens)]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(news), max(need)), -1)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = order[at:at + k]
            at += k
        self.ref = kvref.RefCache(pages, heads, dim, page, kb, vb, rng)
        self.news, self.lens, self.tokens = news, lens, sum(news)
        self.starts = np.concatenate([[0], np.cumsum(news)])
        kbuf, vbuf = self.ref.buffers()
        self.cache = d.KVCache(dev(kbuf), dev(vbuf), pages, heads, dim, page, ENC[kb], ENC[vb])
        self.batch = self.kv_batch(news)

    def kv_batch(self, news, lens=None):
        lens = self.lens if lens is None else lens
        starts = np.concatenate([[0], np.cumsum(news)])
        return d.KVBatch(i32(self.table), i32(lens), i32(starts), int(sum(news)), int(max(news)),
                         int(max(a + b for a, b in zip(news, lens))))

    def same_bytes(self):
        kb, vb = self.ref.buffers()
        # every NaN scale is the same NaN
        return np.array_equal(self.cache.k.cpu().numpy(), kb) and np.array_equal(self.cache.v.cpu().numpy(), vb)

    def write(self, k, v):
        """The reference's append of f32 rows (already rotated)."""
        r = self.ref
        kc, ks = kvref.quant(k, r.kb, 32)
        vc, vs = kvref.quant(v, r.vb, r.dim)
        for b, (n, l) in enumerate(zip(self.news, self.lens)):
            for i in range(n):
                p, s, t = self.table[b][(l + i) // r.page], (l + i) % r.page, self.starts[b] + i
                if not 0 <= p < r.pages:
                    continue
                r.kc[p, :, s], r.ks[p, :, s] = kc[t], ks[t]
                r.vc[p, :, s], r.vs[p, :, s] = vc[t], vs[t, :, 0]


def rows(rng, tokens, heads, dim, dtype, how):
    """Random rows as a device tensor: contiguous, a slice of a fused one, off 16-byte boundaries, or head-major."""
    x = rng.normal(0, 1, (tokens, heads, dim)).astype(np.float32)
    x *= np.where(rng.random((1, heads, dim)) < 0.05, 8, 1)
    t = dev(x, dtype)
    if how == "fused":
        wide = torch.zeros((tokens, heads + 3, dim), dtype=dtype, device="cuda")
        wide[:, 2:2 + heads] = t
        t = wide[:, 2:2 + heads]
    elif how == "odd":
        flat = torch.zeros(tokens * (heads * dim + 1) + 1, dtype=dtype, device="cuda")[1:]
        v = flat.as_strided((tokens, heads, dim), (heads * dim + 1, dim, 1))
        v.copy_(t)
        t = v
    elif how == "head_major":
        t = t.transpose(0, 1).contiguous().transpose(0, 1)
    return t, t.float().cpu().numpy()


HOW = ["plain", "fused", "odd", "head_major"]


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("kb,vb", [(8, 8), (8, 4), (4, 8), (4, 4)])
@pytest.mark.parametrize("page,news,lens", [
    (16, [1], [0]), (16, [1, 1, 1], [15, 16, 4097]), (32, [3, 0, 17, 40], [5, 9, 0, 30]), (64, [2, 70], [127, 3]),
    (256, [33, 16, 5], [250, 16, 12])])
def test_append_bytes(ctx, dim, kb, vb, page, news, lens):
    c = Case(dim + kb + vb, news, lens, 3, dim, page, kb, vb)
    dtype = DT["bf16" if (dim // 32 + kb) % 2 else "f32"]
    k, kf = rows(c.rng, c.tokens, 3, dim, dtype, HOW[(page // 16 + vb) % 4])
    v, vf = rows(c.rng, c.tokens, 3, dim, dtype, HOW[(page // 16 + kb) % 4])
    assert ctx.kv_append(c.cache, c.batch, k, v) is None
    c.write(kf, vf)
    assert c.same_bytes()


@pytest.mark.parametrize("bits", [8, 4])
def test_append_special_values(ctx, bits):
    """Zeros, ties of magnitude, exact halves, subnormals, the largest numbers, infinities and NaN."""
    c = Case(5, [16], [0], 1, 64, 16, bits, bits)
    x = np.zeros((16, 1, 64), np.float32)
    x[1] = 1.0
    x[2, 0, :32] = np.linspace(-1, 1, 32)  # the extremes tie
    x[3] = np.arange(64) / 2 * (127.0 / 31.5)
    x[4] = 1e-40 * np.arange(64)
    x[5] = 3.4e38 * np.where(np.arange(64) % 2, 1, -1)
    x[6, 0, 3] = np.inf
    x[7, 0, 40] = -np.inf
    x[8, 0, 0] = np.nan
    x[9] = 1e-45
    x[10] = np.where(np.arange(64) % 3, -0.0, 0.0)
    x[11, 0, 63] = -7.25
    x[12, 0, 0] = 127.5
    x[12, 0, 1:] = np.arange(1, 64) - 0.5
    t = dev(x)
    ctx.kv_append(c.cache, c.batch, t, t)
    before = c.ref.copy()
    c.write(x, x)
    kb, vb = c.ref.buffers()
    # a scale of zero may carry either sign
    got_k, got_v = c.cache.k.cpu().numpy(), c.cache.v.cpu().numpy()
    n_k, n_v = c.ref.kc.size * bits // 8, c.ref.vc.size * bits // 8
    assert np.array_equal(got_k[:n_k], kb[:n_k]) and np.array_equal(got_v[:n_v], vb[:n_v])
    val = lambda a, n: torch.from_numpy(a[n:].copy()).view(torch.bfloat16).float().numpy()
    np.testing.assert_array_equal(val(got_k, n_k), val(kb, n_k))
    np.testing.assert_array_equal(val(got_v, n_v), val(vb, n_v))
    back, _ = ctx.kv_read(c.cache, c.batch)
    back = back.cpu().numpy()
    assert np.isnan(back[6, 0, :32]).all() and np.isfinite(back[6, 0, 32:]).all()
    assert np.isnan(back[7, 0, 32:]).all() and np.isfinite(back[7, 0, :32]).all()
    assert before.pages == c.ref.pages


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (128, 32), (96, 96), (96, 24), (256, 256), (64, 2), (128, 20), (256, 80)])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_append_rotates_keys_and_queries(ctx, layout, dim, rot, io):
    c = Case(rot, [5, 19], [40, 3], 2, dim, 32, 8, 8)
    tab = kvref.table(64, rot).astype(np.float32)
    pos = c.rng.integers(0, 64, c.tokens)
    pos[3] = 64  # beyond the table
    pos[7] = -1
    k, kf = rows(c.rng, c.tokens, 2, dim, DT[io], "fused")
    v, vf = rows(c.rng, c.tokens, 2, dim, DT[io], "plain")
    q, qf = rows(c.rng, c.tokens, 6, dim, DT[io], "odd" if rot == 32 else "fused")
    rope = d.Rope(dev(tab), i32(pos), rot, layout)
    out = ctx.kv_append(c.cache, c.batch, k, v, rope=rope, q=q)
    turned = kvref.rotate(qf, tab, pos, rot, layout == "half")
    np.testing.assert_array_equal(out.float().cpu().numpy(), turned if io == "f32" else kvref.bf16(turned))
    c.write(kvref.rotate(kf, tab, pos, rot, layout == "half"), vf)
    assert c.same_bytes()
    # the same rotation by itself, into a new tensor and in place
    alone = ctx.rope(q, rope)
    assert torch.equal(alone.view(torch.uint8), out.view(torch.uint8))
    assert ctx.rope(q, rope, out=q) is q
    assert torch.equal(q.contiguous().view(torch.uint8), out.contiguous().view(torch.uint8))


@pytest.mark.parametrize("scaling,kw", [
    ("none", {}), ("linear", dict(factor=8.0)), ("yarn", dict(factor=16.0, original=4096.0)),
    ("yarn", dict(factor=4.0, original=8192.0, attn=1.5, fast=20.0, slow=2.0)),
    ("bands", dict(factor=8.0, original=8192.0, low=1.0, high=4.0))])
@pytest.mark.parametrize("rot,theta", [(128, 1e6), (24, 1e4), (2, 10.0)])
def test_rope_table(ctx, scaling, kw, rot, theta):
    names = dict(factor="factor", original="original_length", attn="attn_factor", fast="beta_fast", slow="beta_slow",
                 low="low_turns", high="high_turns")
    n = 70001
    got = ctx.rope_table(n, rot, theta, scaling, **{names[k]: v for k, v in kw.items()}).cpu().numpy()
    ref = kvref.table(n, rot, theta, scaling, **kw)
    # one f32 rounding of values up to 1.5; the 64-bit angles (up to 7e4) agree to 7e4 * 2^-50
    assert np.abs(got - ref).max() <= 1.5 * 2.0 ** -24 + 1e-10
    assert ctx.rope_table(0, rot, theta).shape == (0, rot // 2, 2)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("kb,vb", [(8, 4), (4, 8)])
@pytest.mark.parametrize("page,news,lens", [(16, [1], [0]), (16, [50, 0, 3], [7, 3, 31]), (128, [200, 16], [100, 16])])
def test_read_back(ctx, dim, kb, vb, page, news, lens):
    c = Case(dim, news, lens, 4, dim, page, kb, vb)
    want = [np.concatenate([c.ref.rows(c.table[b], l, n, kind) for b, (n, l) in enumerate(zip(news, lens))])
            for kind in "kv"]
    k, v = ctx.kv_read(c.cache, c.batch)
    np.testing.assert_array_equal(k.cpu().numpy(), want[0])
    np.testing.assert_array_equal(v.cpu().numpy(), want[1])
    k, v = ctx.kv_read(c.cache, c.batch, dtype=torch.bfloat16)
    np.testing.assert_array_equal(k.float().cpu().numpy(), kvref.bf16(want[0]))
    np.testing.assert_array_equal(v.float().cpu().numpy(), kvref.bf16(want[1]))
    for how in ("fused", "odd", "head_major"):  # either alone, into strided rows
        out, _ = rows(c.rng, c.tokens, 4, dim, torch.float32, how)
        ctx.kv_read(c.cache, c.batch, v_out=out)
        np.testing.assert_array_equal(out.cpu().numpy(), want[1])
        ctx.kv_read(c.cache, c.batch, k_out=out)
        np.testing.assert_array_equal(out.cpu().numpy(), want[0])


@pytest.mark.parametrize("kb,vb", [(8, 8), (4, 4)])
def test_absent_pages(ctx, kb, vb):
    """Page ids out of range and positions beyond the table: nothing is written, NaN is read."""
    c = Case(3, [40, 40], [0, 20], 2, 64, 16, kb, vb)
    c.table[0, 1], c.table[1, 2] = -7, c.ref.pages
    c.table = np.ascontiguousarray(c.table[:, :3])  # sequence 1 runs beyond it
    c.batch = c.kv_batch(c.news)
    k, kf = rows(c.rng, 80, 2, 64, torch.float32, "plain")
    v, vf = rows(c.rng, 80, 2, 64, torch.float32, "plain")
    ctx.kv_append(c.cache, c.batch, k, v)
    c.table = np.concatenate([c.table, np.full((2, 1), -1)], 1)
    c.write(kf, vf)
    assert c.same_bytes()
    got, _ = ctx.kv_read(c.cache, c.batch)
    want = np.concatenate([c.ref.rows(c.table[b], l, 40, "k") for b, l in enumerate([0, 20])])
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    assert np.isnan(want).any()


def test_tables_out_of_range(ctx):
    """Starts beyond the rows or out of order, more rows than max_new, a negative length."""
    c = Case(4, [6, 6, 6], [0, 4, 9], 2, 64, 16, 8, 4)
    k, kf = rows(c.rng, 18, 2, 64, torch.float32, "plain")
    batch = d.KVBatch(i32(c.table), i32([0, -3, 9]), i32([0, 6, 3, 99]), 18, 4, 20)
    ctx.kv_append(c.cache, batch, k, k)
    c.news, c.lens, c.starts = [4, 0, 4], [0, 0, 9], [0, 6, 3]
    c.write(kf, kf)
    assert c.same_bytes()


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("kb,vb", [(8, 8), (8, 4), (4, 8), (4, 4)])
@pytest.mark.parametrize("page", [16, 64])
def test_commit(ctx, dim, kb, vb, page):
    news, lens = [9, 24, 1, 40, 0], [0, 13, 5, 60, 3]
    c = Case(dim + page, news, lens, 2, dim, page, kb, vb)
    width = 24
    path, counts = np.full((5, width), -1), np.zeros(5, int)
    for b, n in enumerate(news):
        p = sorted({0} | set(c.rng.choice(n, size=min(n, width) // 2 + 1).tolist())) if n else []
        counts[b] = len(p)
        path[b, :len(p)] = p
    ref = c.ref
    ctx.kv_commit(c.cache, c.batch, i32(path), i32(counts))
    for b, l in enumerate(lens):
        for j in range(counts[b]):
            src, dst = l + path[b, j], l + j
            ps, ss, pd, sd = c.table[b][src // page], src % page, c.table[b][dst // page], dst % page
            for a in (ref.kc, ref.ks, ref.vc, ref.vs):
                a[pd, :, sd] = a[ps, :, ss]
    assert c.same_bytes()
    # entries that do not ascend, or lie outside the rows, are left out
    ctx.kv_commit(c.cache, c.batch, i32(np.where(path < 0, -1, 0)), i32(np.full(5, 99)))
    ctx.kv_commit(c.cache, c.batch, i32(np.full((5, width), 4000)), i32(np.full(5, width)))
    assert c.same_bytes()


def test_empty_calls(ctx):
    c = Case(1, [1], [0], 1, 64, 16, 8, 8)
    none = torch.empty((0, 1, 64), device="cuda")
    batch = d.KVBatch(i32(c.table), i32([0]), i32([0, 0]), 0, 0, 0)
    ctx.kv_append(c.cache, batch, none, none)
    assert ctx.kv_read(c.cache, batch)[0].shape == (0, 1, 64)
    ctx.kv_commit(c.cache, batch, torch.empty((1, 0), dtype=torch.int32, device="cuda"), i32([0]))
    assert ctx.tree_attention(c.cache, batch, none).shape == (0, 1, 64)
    no_seq = d.KVBatch(torch.empty((0, 4), dtype=torch.int32, device="cuda"), i32([]), i32([0]), 0, 0, 0)
    ctx.kv_append(c.cache, no_seq, none, none)
    assert c.same_bytes()


def test_other_stream_and_graph(ctx):
    """On a stream of its own and captured: replays write and read the same bytes."""
    c = Case(8, [4, 20], [30, 7], 2, 128, 32, 8, 4)
    k, kf = rows(c.rng, c.tokens, 2, 128, torch.bfloat16, "fused")
    v, vf = rows(c.rng, c.tokens, 2, 128, torch.bfloat16, "fused")
    kb, vb = torch.empty((2, c.tokens, 2, 128), device="cuda").unbind(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ctx.kv_append(c.cache, c.batch, k, v, stream=s)
    a, b = ctx.kv_read(c.cache, c.batch, stream=s)
    s.synchronize()
    c.write(kf, vf)
    assert c.same_bytes()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.kv_append(c.cache, c.batch, k, v)
        ctx.kv_read(c.cache, c.batch, k_out=kb, v_out=vb)
    for _ in range(3):
        c.cache.k.zero_(), kb.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(kb, a) and torch.equal(vb, b)


def bad(fn, code=d.ERR_INVALID_ARGUMENT):
    with pytest.raises(d.DyninferError) as e:
        fn()
    assert e.value.code == code


def test_refusals(ctx):
    c = Case(2, [4], [0], 2, 64, 16, 8, 8)
    x = torch.zeros((4, 2, 64), device="cuda")
    tab, pos = dev(kvref.table(8, 64).astype(np.float32)), i32([0, 1, 2, 3])
    rope = d.Rope(tab, pos, 64)
    app = lambda k=x, v=x, cache=c.cache, batch=c.batch, **kw: ctx.kv_append(cache, batch, k, v, **kw)
    over = lambda **kw: d.KVCache(**{**c.cache.__dict__, **kw})
    bad(lambda: app(k=x.cpu()))
    bad(lambda: app(k=x[:3]))
    bad(lambda: app(k=torch.zeros((4, 64, 2), device="cuda").transpose(1, 2)))
    bad(lambda: app(k=x.bfloat16()))                      # k and v differ
    bad(lambda: app(k=x.half(), v=x.half()), d.ERR_UNSUPPORTED)
    bad(lambda: app(k=x[:, :1], v=x[:, :1]))              # not the cache's heads
    bad(lambda: app(q=x))                                 # no rope
    bad(lambda: app(rope=rope, q=x, q_out=x[:, :1]))
    bad(lambda: app(rope=rope, q=x, q_out=torch.zeros((1, 2, 64), device="cuda").expand(4, 2, 64)))
    bad(lambda: app(rope=rope, q=torch.zeros_like(x), q_out=x))  # q_out is k
    bad(lambda: app(rope=d.Rope(tab, pos, 66)))
    bad(lambda: app(rope=d.Rope(tab, pos[:2], 64)))
    bad(lambda: app(rope=d.Rope(tab, pos, 64, "other")))
    bad(lambda: app(cache=over(pages=c.cache.pages + 1)))
    bad(lambda: app(cache=over(k=c.cache.k[16:])))
    bad(lambda: app(cache=over(k_encoding=3)), d.ERR_UNSUPPORTED)
    bad(lambda: app(cache=over(head_dim=80)))             # the rows do not fit it
    bad(lambda: d.KVCache.bytes(4, 2, 80), d.ERR_UNSUPPORTED)
    bad(lambda: d.KVCache.bytes(4, 2, 64, page_size=48), d.ERR_UNSUPPORTED)
    bad(lambda: d.KVCache.bytes(4, 2, 64, page_size=8), d.ERR_UNSUPPORTED)
    bad(lambda: d.KVCache.bytes(0, 2, 64))
    bad(lambda: d.KVCache.bytes(4, -2, 64))
    over_b = lambda **kw: d.KVBatch(**{**c.batch.__dict__, **kw})
    bad(lambda: app(batch=over_b(max_new=5)))
    bad(lambda: app(batch=over_b(starts=i32([0, 2, 4]))))
    bad(lambda: app(batch=over_b(lengths=torch.zeros(1, dtype=torch.int64, device="cuda"))))
    bad(lambda: app(batch=over_b(page_table=c.batch.page_table.cpu())))
    bad(lambda: ctx.kv_read(c.cache, c.batch, k_out=x, v_out=x))
    bad(lambda: ctx.kv_read(c.cache, c.batch, k_out=x[:, :1].expand(4, 2, 64)))
    bad(lambda: ctx.kv_commit(c.cache, c.batch, pos[None], i32([1, 1])))
    bad(lambda: ctx.rope(x, d.Rope(tab, pos, 63)))
    bad(lambda: ctx.rope(x, rope, out=x.view(-1)[:256].view(4, 1, 64).expand(4, 2, 64)))
    bad(lambda: ctx.rope(torch.zeros((4, 2, 80), device="cuda"), rope), d.ERR_UNSUPPORTED)
    bad(lambda: ctx.rope_table(8, 64, scaling="other"))
    bad(lambda: ctx.rope_table(8, 64, theta=0.5))
    bad(lambda: ctx.rope_table(8, 64, scaling="yarn", factor=2.0))
    bad(lambda: ctx.rope_table(8, 64, scaling="bands", factor=2.0, original_length=4096.0, low_turns=4.0, high_turns=1.0))
    assert c.same_bytes()


@pytest.mark.parametrize("rot", [8, 24, 40, 64, 72, 96])
def test_rope_outside_the_table(ctx, rot):
    """Positions on both sides of a short table: NaN in the rotated dims, the rest kept."""
    x = torch.randn((5, 3, 96), device="cuda")
    table = ctx.rope_table(2, rot)
    pos = i32([0, -1, 1, 2, 2 ** 31 - 1])
    for layout in ("half", "interleaved"):
        y = ctx.rope(x, d.Rope(table, pos, rot, layout))
        assert torch.equal(y[:, :, rot:], x[:, :, rot:])
        assert torch.isnan(y[:, :, :rot]).all(-1).all(-1).tolist() == [False, True, False, True, True]
        assert not torch.isnan(y[[0, 2]]).any()


def test_commit_of_paths_without_entries(ctx):
    """What verification returns where no sequence may have rows: paths of width 0 move nothing."""
    c = Case(30, [5, 3], [7, 20], 2, 64, 16, 8, 4)
    for counts in ([0, 0], [2, 1]):
        ctx.kv_commit(c.cache, c.batch, torch.empty((2, 0), dtype=torch.int32, device="cuda"), i32(counts))
    assert c.same_bytes()


def test_sequences_without_pages(ctx):
    """A page table of no columns: every position is absent."""
    c = Case(31, [2, 1], [0, 5], 2, 64, 16, 8, 8)
    batch = d.KVBatch(torch.empty((2, 0), dtype=torch.int32, device="cuda"), c.batch.lengths, c.batch.starts, 3, 2, 6)
    k, v, q = (torch.randn((3, h, 64), device="cuda") for h in (2, 2, 4))
    table = ctx.rope_table(8, 64)
    pos = i32([0, 1, 5])
    got = ctx.kv_append(c.cache, batch, k, v, rope=d.Rope(table, pos, 64), q=q)
    assert torch.equal(got, ctx.rope(q, d.Rope(table, pos, 64))) and c.same_bytes()
    assert all(torch.isnan(x).all() for x in ctx.kv_read(c.cache, batch))
    lse = torch.zeros((3, 4), device="cuda")
    assert (ctx.tree_attention(c.cache, batch, q, lse=lse) == 0).all() and (lse == -float("inf")).all()
    ctx.kv_commit(c.cache, batch, i32([[0, 1], [0, -1]]), i32([2, 1]))
    assert c.same_bytes()
    none = d.KVBatch(batch.page_table, batch.lengths, i32([0, 0, 0]), 0, 0, 5)  # nor rows
    ctx.kv_append(c.cache, none, k[:0], v[:0])
    assert all(x.shape == (0, 2, 64) for x in ctx.kv_read(c.cache, none))


@pytest.mark.parametrize("call", ["append", "read", "commit", "attend"])
def test_calls_of_too_many_threads(ctx, call):
    """A launch's threads are counted in 32 bits: calls that need more are refused as such, smaller ones run."""
    n = 1 << 20
    zero = torch.zeros((n, 1), dtype=torch.int32, device="cuda")
    starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    starts[-1] = 1  # the last sequence has a row
    batch = d.KVBatch(zero, zero[:, 0].contiguous(), starts, 1, 1, 1)

    def run(heads):
        cache = d.KVCache.empty(1, heads, 64, 16)
        x = torch.randn((1, heads, 64), device="cuda")
        ctx.kv_append(cache, d.KVBatch(zero[:1], zero[0], i32([0, 1]), 1, 1, 1), x, x)
        if call == "append":
            ctx.kv_append(cache, batch, x, x)
        elif call == "read":
            return ctx.kv_read(cache, batch)[1], x
        elif call == "commit":
            ctx.kv_commit(cache, batch, zero, zero[:, 0].contiguous())
        else:
            return ctx.tree_attention(cache, batch, x), x
        return ctx.kv_read(cache, d.KVBatch(zero[:1], zero[0], i32([0, 1]), 1, 1, 1))[1], x

    bad(lambda: run(64), d.ERR_UNSUPPORTED)
    got, x = run(1)
    # a value's code is at most half a scale off, the scale that of the largest / 127, rounded to 8 bits
    assert (got - x).abs().max() <= x.abs().max() * (0.5 / 127 + 2 ** -8) * 1.01
