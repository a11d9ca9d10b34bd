"""Log probabilities, ranks, entropy and alternatives on the GPU, against 64 bits.  Ranks and
tokens are equal; of what is computed the tolerance is, in units of 2^-24 (one rounding):

a power e^t with t = (x - m) / T: t has the roundings of the difference, of 1 / T twice, of the
product and the exponential's two: 4 |t| + 2; a sum of a row: 32 terms a thread, 6 + 2 steps of joining, then
256 threads over the pieces, 8 more steps, so 50 with pieces / 256 on top.  So ln S is off by 52 + 4 sum p |t|
+ 2 |ln S|, t by 4 |t|, U / S by 2 * 52 |U / S| + 4 sum p t^2 + 6 sum p |t|."""
import numpy as np
import pytest
import torch

import dyninfer_amd as d

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
U = 2.0**-24


def plain(x):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    return np.minimum(x, float(np.finfo(np.float32).max))


def check(got, x, tokens, top, temperature=None):
    """got: TokenLogprobs; x: f32 array [rows, vocab] of the logits as the call saw them."""
    lp, rk, en, tt, tl = [None if t is None else t.cpu().numpy() for t in got]
    for r in range(len(x)):
        v = plain(x[r])
        order = np.argsort(-v, kind="stable")
        temp = 1.0 if temperature is None else float(temperature[r])
        m = v[order[0]]
        some = m > -np.inf
        with np.errstate(invalid="ignore", over="ignore"):
            t = np.where(v > -np.inf, v - m, -np.inf) if some else np.full_like(v, -np.inf)
        if temp > 0:
            t = np.where(t > -np.inf, t / temp, -np.inf)
            e = np.exp(t)
            s = e.sum() if some else 1.0
            p = e / s
            tp = np.where(e > 0, t, 0.0)
            a1, a2 = (p * -tp).sum(), (p * tp * tp).sum()
            logp = t - np.log(s)
            tol_s = U * (52 + len(v) / 8192 / 256 + 4 * a1 + 2 * np.log(s))
            tol = np.where(t > -np.inf, tol_s + U * (4 * np.abs(t) + np.abs(logp)), 0.0) + 1e-38
            h, tol_h = (np.log(s) + a1 if some else 0.0), tol_s + U * (110 * a1 + 4 * a2 + 6 * a1) + 1e-38
        else:
            logp = np.where(np.arange(len(v)) == order[0], 0.0, -np.inf) if some else t
            tol, h, tol_h = np.zeros_like(v), 0.0, 0.0

        def near(y, i):
            assert (y == logp[i]) if np.isinf(logp[i]) or np.isinf(y) else abs(y - logp[i]) <= tol[i], (r, i, y, logp[i], tol[i])

        assert abs(en[r] - h) <= tol_h, (r, en[r], h, tol_h)
        if tokens is not None:
            k = int(tokens[r])
            if 0 <= k < len(v):
                assert rk[r] == int(np.nonzero(order == k)[0][0]), (r, k)
                near(lp[r], k)
            else:
                assert rk[r] == -1 and lp[r] == -np.inf
        if top:
            best = [k for k in order[:top] if v[k] > -np.inf]
            assert tt[r].tolist() == best + [-1] * (top - len(best)), r
            for i, k in enumerate(best):
                near(tl[r, i], k)
            assert (tl[r, len(best):] == -np.inf).all()


def case(seed, n, vocab, io, how="plain", spread=2.5):
    """Logits as a device tensor (rows at any boundary, with a stride) and as the call sees them."""
    rng = np.random.default_rng(seed)
    x = rng.normal(0, spread, (n, vocab)).astype(np.float32)
    t = torch.from_numpy(x).cuda().to(DT[io])
    if how != "plain":
        off, stride = {"odd": (1, vocab + 1), "far": (3, vocab + 1000)}[how]
        flat = torch.full((off + n * stride,), float("nan"), dtype=DT[io], device="cuda")
        v = flat[off:].as_strided((n, vocab), (stride, 1))
        v.copy_(t)
        t = v
    return rng, t, t.float().cpu().numpy()


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 63, 64, 65, 300, 8185, 8191, 8192, 8193, 8200, 16384, 32003, 151936])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("n,top,how", [(1, 20, "plain"), (3, 5, "odd"), (5, 0, "far"), (2, 64, "odd")])
def test_sizes(ctx, vocab, io, n, top, how):
    rng, t, x = case(vocab + n, n, vocab, io, how)
    tokens = rng.integers(0, vocab, n)
    tokens[0] = (0, vocab - 1, int(np.argmax(x[0])))[top % 3]
    got = ctx.token_logprobs(t, torch.from_numpy(tokens).cuda(), top=top)
    check(got, x, tokens, top)


def test_many_pieces(ctx):
    """More pieces than a workgroup has threads."""
    rng, t, x = case(1, 2, (1 << 21) + 20005, "bf16", "odd")
    tokens = np.array([(1 << 21) + 20004, 8192 * 256])
    check(ctx.token_logprobs(t, torch.from_numpy(tokens).cuda(), top=33), x, tokens, 33)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["equal", "two", "up", "down", "few", "one", "none", "zeros", "steps"])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_ties_and_masks(ctx, io, kind, top):
    vocab = 20011
    rng, t, x = case(7, 2, vocab, io, "odd")
    if kind == "equal":
        t.fill_(1.5)
    elif kind == "two":  # two values
        t.copy_((t > 0).to(t.dtype))
    elif kind in ("up", "down"):
        y = torch.linspace(-9, 9, vocab, device="cuda").to(t.dtype)
        t.copy_(y if kind == "up" else y.flip(0))
    elif kind in ("few", "one", "none"):
        keep = torch.zeros(2, vocab, dtype=torch.bool, device="cuda")
        keep[:, torch.from_numpy(rng.choice(vocab, {"few": 11, "one": 1, "none": 1}[kind], replace=False)).cuda()] = kind != "none"
        t.masked_fill_(~keep, float("-inf"))
    elif kind == "zeros":  # 0 and -0 tie
        t.copy_(torch.where(t > 0, 0.0, -0.0).to(t.dtype))
    else:  # one thread's logits are the largest
        t[:, 8000:8040] += 50.0
    x = t.float().cpu().numpy()
    for k in (0, 8005, vocab - 1, int(rng.integers(vocab))):
        tokens = np.array([k, (k + 9000) % vocab])
        check(ctx.token_logprobs(t, torch.from_numpy(tokens).cuda(), top=top), x, tokens, top)


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_special_logits(ctx, io):
    vocab = 9001
    rng, t, _ = case(11, 9, vocab, io)
    big = float(torch.finfo(DT[io]).max)
    t[0, 5] = float("inf")
    t[1, 5], t[1, 8500] = float("inf"), float("inf")
    t[2, ::3] = float("nan")
    t[3, 7:] = float("nan")
    t[4] = float("nan")
    t[5, 17], t[5, 18] = float("inf"), big
    t[6, 100] = -big
    t[6, 101] = float("-inf")
    t[7] *= 1e30
    t[8, 0], t[8, 1], t[8, 2:] = 3.0, float("nan"), float("-inf")
    x = t.float().cpu().numpy()
    for tokens in ([5, 8500, 3, 7, 9, 18, 101, 4, 1], [17, 5, 1, 2, 0, 17, 100, 0, 0], [9000] * 9):
        got = ctx.token_logprobs(t, torch.tensor(tokens, device="cuda"), top=9)
        assert not any(torch.isnan(g).any() for g in (got.logprobs, got.entropy, got.top_logprobs))
        check(got, x, tokens, 9)


def test_temperatures(ctx):
    vocab, io = 5000, "f32"
    temps = [0.0, 1.0, 0.3, 7.0, -1.0, 1e-3, 1e4, 1e-30, 1e36, 2.0**-20, -float("inf"), 0.7]
    rng, t, _ = case(13, len(temps), vocab, io)
    t[11, 50:] = float("-inf")
    x = t.float().cpu().numpy()
    tokens = np.array([int(np.argmax(v)) if i % 3 else 77 for i, v in enumerate(x)])
    temperature = torch.tensor(temps, dtype=torch.float32, device="cuda")
    check(ctx.token_logprobs(t, torch.from_numpy(tokens).cuda(), top=12, temperature=temperature), x, tokens, 12,
          np.array(temps, np.float32))
    # beyond the range: as the largest and the smallest one; NaN: NaN
    t = t[:4].clone()
    t[2, 100:] = float("-inf")
    got = ctx.token_logprobs(t, top=3, temperature=torch.tensor([float("inf"), 1e-45, float("inf"), float("nan")], device="cuda"))
    assert abs(got.entropy[0].item() - np.log(vocab)) < 1e-5 and got.entropy[1].item() == 0.0
    assert abs(got.entropy[2].item() - np.log(100)) < 1e-5
    assert got.top_logprobs[1, 0] == 0.0 and (got.top_logprobs[1, 1:] < -1e34).all()
    assert torch.isnan(got.entropy[3]) and torch.isnan(got.top_logprobs[3]).all()


def test_tokens_outside(ctx):
    vocab = 301
    _, t, x = case(17, 6, vocab, "bf16")
    tokens = np.array([-1, vocab, -100, 2**40, 300, 0])
    got = ctx.token_logprobs(t, torch.from_numpy(tokens).cuda(), top=2)
    check(got, x, tokens, 2)


def test_what_is_asked_for(ctx):
    _, t, x = case(19, 4, 1000, "f32")
    got = ctx.token_logprobs(t)
    assert got.logprobs is None and got.ranks is None and got.top_tokens is None and got.top_logprobs is None
    check(got, x, None, 0)
    empty = ctx.token_logprobs(t[:0], torch.empty(0, dtype=torch.int64, device="cuda"), top=3)
    assert empty.entropy.shape == (0,) and empty.top_tokens.shape == (0, 3)
    # one row shown to several: a stride of 0 is refused, a copy is not
    with pytest.raises(d.DyninferError):
        ctx.token_logprobs(t[:1].expand(3, -1))
    check(ctx.token_logprobs(t[:1].expand(1, -1), top=64), x[:1], None, 64)


def test_same_every_time_and_in_a_graph(ctx):
    _, t, _ = case(23, 40, 30000, "bf16", "odd")
    tokens = torch.randint(0, 30000, (40,), device="cuda")
    first = ctx.token_logprobs(t, tokens, top=7)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ctx.token_logprobs(t, tokens, top=7)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ctx.token_logprobs(t, tokens, top=7, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ctx.token_logprobs(t, tokens, top=7)
    for _ in range(3):
        t.copy_(torch.randn(40, 30000, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ctx.token_logprobs(t, tokens, top=7)))


def test_rows_beyond_32_bits(ctx):
    """Rows whose offsets pass 2^32 elements."""
    vocab, stride = 1000, (1 << 31) + 9
    flat = torch.empty(2 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    t = flat.as_strided((3, vocab), (stride, 1))
    t.copy_(torch.randn(3, vocab, device="cuda"))
    tokens = torch.tensor([0, 999, 5], device="cuda")
    check(ctx.token_logprobs(t, tokens, top=5), t.float().cpu().numpy(), [0, 999, 5], 5)


def test_refused(ctx):
    x, t = torch.zeros(3, 9000, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    good = dict(logits=x, tokens=t, top=2)
    ctx.token_logprobs(**good)
    for bad in (dict(logits=x[0]), dict(logits=x.cpu()), dict(logits=x.half()), dict(logits=x[:, ::2]), dict(logits=x.double()[:, :9]),
                dict(logits=x[:1].expand(3, 9000)), dict(logits=x[:, :0]), dict(tokens=t[:2]), dict(tokens=t.int()), dict(tokens=t.cpu()),
                dict(top=65), dict(top=-1), dict(top=1 << 40), dict(top=1.5), dict(temperature=torch.ones(2, device="cuda")),
                dict(temperature=torch.ones(3, device="cuda").double()), dict(workspace=torch.empty(16, device="cuda"))):
        with pytest.raises((d.DyninferError, TypeError)):
            ctx.token_logprobs(**{**good, **bad})
