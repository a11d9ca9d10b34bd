"""The operators that a prompt needs around its quantised products, and how their speed is measured.

A program that reads a prompt, to answer it or to score a text, needs of every layer: the norm of
each query and key head with the position rotation (models that normalise them have it between the
projection and the attention; on the way into the quantised cache for the tokens that are decoded
one by one), and causal attention over the prompt's own keys and values, before they are rounded to
a cache's codes; and at the end, of the logits, the log probability of the tokens that came, its
rank, the distribution's entropy and the likeliest alternatives.

Cases name the operator in ``op``.  Rows of a call are tokens packed sequence after sequence; in
attention a sequence has as many keys as rows, or more: then its rows are the last ones.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False  # False: the plain forms; True: the framework's kernels

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
VOCAB = 151936
POSITIONS = 32768
EPS = 1e-6


def listed():
    return [
        # One token of the small model: a call that is all latency.
        dict(name="qk_1token", op="qk", tokens=1, q_heads=16, kv_heads=8, dim=128, rot=128, layout="half", io="bf16",
             weight="bf16", offset=0.0, fused=True),
        # A middling prompt in f32, a part of each head rotated, weights kept as differences from one.
        dict(name="qk_517_f32", op="qk", tokens=517, q_heads=20, kv_heads=5, dim=96, rot=64, layout="interleaved",
             io="f32", weight="f32", offset=1.0, fused=False),
        # A long prompt of the large model, slices of one fused projection.
        dict(name="qk_prompt_8191", op="qk", tokens=8191, q_heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             io="bf16", weight="f32", offset=0.0, fused=True),
        # A decoding step of thirty-two sequences: norm, rotation, the keys and values into the cache; read back.
        dict(name="append_32x1", op="append", seqs=32, new=1, ragged=0, length=700, q_heads=32, kv_heads=8, dim=128,
             rot=128, layout="half", v="q8", page=64, io="bf16", weight="bf16", offset=0.0),
        # A short prompt of the small model in f32.
        dict(name="attend_1x37_f32", op="attend", seqs=1, new=37, ragged=0, prior=0, q_heads=16, kv_heads=8, dim=128,
             io="f32", fused=True),
        # Twenty-four prompts of different lengths packed together.
        dict(name="attend_24x1000", op="attend", seqs=24, new=1000, ragged=1, prior=0, q_heads=16, kv_heads=8, dim=128,
             io="bf16", fused=True),
        # Pieces of two long prompts after what was read before, small heads: few rows, many keys.
        dict(name="attend_2x96_after_24k", op="attend", seqs=2, new=96, ragged=2, prior=24000, q_heads=12, kv_heads=4,
             dim=64, io="bf16", fused=False),
        # Three prompts in f32 with wide heads.
        dict(name="attend_3x1500_f32", op="attend", seqs=3, new=1500, ragged=3, prior=0, q_heads=8, kv_heads=2, dim=256,
             io="f32", fused=False),
        # One long document.
        dict(name="attend_1x16384", op="attend", seqs=1, new=16384, ragged=0, prior=0, q_heads=32, kv_heads=8, dim=128,
             io="bf16", fused=True),
        # The token that was just drawn, with twenty alternatives.
        dict(name="logprobs_1", op="logprobs", rows=1, vocab=VOCAB, top=20, io="f32", warm=False, masked=False),
        # A batch of decoded tokens with temperatures, some rows under a grammar that allows few tokens.
        dict(name="logprobs_33", op="logprobs", rows=33, vocab=32003, top=8, io="f32", warm=True, masked=True),
        # A text scored token by token.
        dict(name="logprobs_2047", op="logprobs", rows=2047, vocab=VOCAB, top=5, io="bf16", warm=False, masked=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk", "qk", "append", "attend", "attend", "attend", "attend", "logprobs", "logprobs", "logprobs"])
    io = rng.choice(["f32", "bf16"])
    if op == "logprobs":
        c = dict(op=op, rows=_log(rng, 1, 2047), vocab=rng.choice([VOCAB, _log(rng, 300, VOCAB), _log(rng, 300, VOCAB)]),
                 top=rng.choice([0, 1, rng.randint(2, 20), rng.randint(2, 20), rng.randint(21, 64)]), io=io, warm=rng.random() < 0.4,
                 masked=rng.random() < 0.4)
        c["rows"] = max(1, min(c["rows"], 2047 * VOCAB * 2 // (c["vocab"] * _SIZE[io])))
        return c
    dim, kv = rng.choice([64, 96, 128, 128, 256]), _log(rng, 1, 16)
    c = dict(op=op, q_heads=kv * rng.choice([1, 2, 3, 4, 4, 8]), kv_heads=kv, dim=dim, io=io)
    if op == "attend":
        c.update(new=_log(rng, 1, 16384), prior=rng.choice([0, 0, _log(rng, 1, 30000)]), seqs=_log(rng, 1, 64),
                 ragged=rng.choice([0, rng.randint(1, 10**6), rng.randint(1, 10**6)]), fused=rng.random() < 0.5)
        most = 16384 * 16384 * 32 * 128 // (6 if io == "f32" else 1)  # rows * keys * heads * dim
        while c["new"] * (c["new"] + 2 * c["prior"]) * c["q_heads"] * dim > most:
            c["new"], c["prior"] = max(1, c["new"] * 2 // 3), c["prior"] * 2 // 3
        c["seqs"] = max(1, min(c["seqs"], most // (c["new"] * (c["new"] + 2 * c["prior"]) * c["q_heads"] * dim),
                               16384 * 16 * 128 // ((c["new"] + c["prior"]) * kv * dim)))
        return c
    c.update(rot=rng.choice([dim, dim, dim // 2, 24]), layout=rng.choice(["half", "interleaved"]),
             weight=rng.choice(["f32", "bf16"]), offset=rng.choice([0.0, 0.0, 1.0]))
    most = 8191 * 40 * 128 * 2 // (dim * _SIZE[io])
    if op == "qk":
        c.update(tokens=max(1, min(_log(rng, 1, 8191), most // (c["q_heads"] + kv))), fused=rng.random() < 0.5)
        return c
    c.update(seqs=_log(rng, 1, 64), new=_log(rng, 1, 4096), ragged=rng.choice([0, rng.randint(1, 10**6)]),
             length=_log(rng, 1, 16384), v=rng.choice(["q8", "q4"]), page=rng.choice([16, 32, 64, 128, 256]))
    c["new"] = max(1, min(c["new"], most // 2 // (c["seqs"] * (c["q_heads"] + 2 * kv))))
    return c


# ------------------------------------------------------------------ what a case's sizes are
def _sizes(case):
    """New tokens of each sequence and those before them; where they differ, ``ragged`` numbers their choice."""
    rng = random.Random(case["ragged"])
    n, new, top = case["seqs"], case["new"], case.get("prior", case.get("length", 0))
    news = [rng.randint((new + 3) // 4, new) if case["ragged"] else new for _ in range(n)]
    news[rng.randrange(n)] = new
    lens = [rng.randint(top // 4, top) if case["ragged"] else top for _ in range(n)]
    lens[rng.randrange(n)] = top
    return news, lens


def _row_bytes(case):
    """Bytes of one token's K and V of all kv heads in the cache."""
    d = case["dim"]
    return case["kv_heads"] * (d + d // 32 * 2 + d * (8 if case["v"] == "q8" else 4) // 8 + 2)


def work(case):
    op, e = case["op"], _SIZE[case["io"]]
    if op == "logprobs":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * (v * e + 8 + 12 + 12 * case["top"]), "flops": n * v * 7}
    q, kv, d = case["q_heads"], case["kv_heads"], case["dim"]
    if op == "qk":
        t, h = case["tokens"], q + kv
        return {"bytes": t * (2 * h * d * e + case["rot"] * 4 + 4), "flops": t * h * (4 * d + 3 * case["rot"])}
    news, lens = _sizes(case)
    new = sum(news)
    if op == "append":  # q, k, v in; q out; the codes written, read again, their values written in bf16
        row = _row_bytes(case)
        return {"bytes": int(new * ((2 * q + 2 * kv) * d * e + case["rot"] * 4 + 2 * row + 2 * kv * d * 2)),
                "flops": int(new * ((q + kv) * (4 * d + 3 * case["rot"]) + 6 * kv * d))}
    pairs = sum(n * l + n * (n + 1) // 2 for n, l in zip(news, lens))
    return {"bytes": 2 * new * q * d * e + new * q * 4 + 2 * (new + sum(lens)) * kv * d * e, "flops": 4 * pairs * q * d}


# ------------------------------------------------------------------ inputs
def _heads(gen, n, heads, d, key):
    """Projected heads in f32 as norms meet them: rows of different size, keys with a few strong channels."""
    x = torch.randn((n, heads, d), device="cuda", generator=gen) * (0.3 + 2 * torch.rand((n, heads, 1), device="cuda", generator=gen))
    if key:
        x *= torch.where(torch.rand((1, heads, d), device="cuda", generator=gen) < 0.05, 4.0, 1.0)
    return x


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(news):
    return [0] + np.cumsum(news).tolist()


def _inv_freq(rot):
    return 1.0e6 ** (-2.0 * np.arange(rot // 2, dtype=np.float64) / rot)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2654435761 % (1 << 62))
    op, dt = case["op"], _DT[case["io"]]
    st = dict(case=case)
    if op == "logprobs":
        n, v = case["rows"], case["vocab"]
        x = torch.randn((n, v), device="cuda", generator=gen) * 2.5
        x += 7.0 * (torch.rand((n, v), device="cuda", generator=gen) < 8.0 / v)  # a few likely tokens
        tokens = torch.randint(0, v, (n,), device="cuda", generator=gen)
        likely = x.argmax(-1)  # most tokens of a text are likely ones
        tokens = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.6, likely, tokens)
        if case["masked"]:  # a grammar leaves some rows few tokens, down to one
            few = torch.rand((n, 1), device="cuda", generator=gen) < 0.5
            keep = torch.rand((n, v), device="cuda", generator=gen) < 12.0 / v
            keep[torch.arange(n, device="cuda"), likely] = True
            x = x.masked_fill(few & ~keep, float("-inf"))
        st["temperature"] = None
        if case["warm"]:
            st["temperature"] = 0.4 + 1.2 * torch.rand(n, device="cuda", generator=gen)
            st["temperature"][torch.rand(n, device="cuda", generator=gen) < 0.1] = 0.0  # these decode greedily
        st.update(logits=x.to(dt), tokens=tokens)
        return st
    q, kv, d = case["q_heads"], case["kv_heads"], case["dim"]
    if op == "attend":
        news, lens = _sizes(case)
        rows, keys = sum(news), sum(news) + sum(lens)
        a = torch.randn((rows, q, d), device="cuda", generator=gen).to(dt)
        b = torch.randn((keys, kv, d), device="cuda", generator=gen)
        b *= torch.where(torch.rand((1, kv, d), device="cuda", generator=gen) < 0.05, 3.0, 1.0)
        b = b.to(dt)
        c = (torch.randn((keys, kv, d), device="cuda", generator=gen) * (0.3 + torch.rand((keys, kv, 1), device="cuda", generator=gen))).to(dt)
        if case["fused"]:  # slices of one tensor: keys and values of one projection, and the queries where it is theirs too
            if rows == keys:
                w = torch.cat([a, b, c], 1)
                a, b, c = w[:, :q], w[:, q:q + kv], w[:, q + kv:]
            else:
                w = torch.cat([b, c], 1)
                b, c = w[:, :kv], w[:, kv:]
        st.update(q=a, k=b, v=c, news=news, lens=lens, starts=_i32(_starts(news)), scale=d ** -0.5,
                  key_starts=_i32(_starts([n + l for n, l in zip(news, lens)])) if any(lens) else None)
        return st
    if op == "append":
        news, lens = _sizes(case)
        rows = sum(news)
    else:
        rows = case["tokens"]
    wide = torch.cat([_heads(gen, rows, q, d, False), _heads(gen, rows, kv, d, True), _heads(gen, rows, kv, d, False)], 1).to(dt)
    st["q"], st["k"], st["v"] = wide[:, :q], wide[:, q:q + kv], wide[:, q + kv:]
    if op == "qk" and not case["fused"]:
        st["q"], st["k"] = st["q"].contiguous(), st["k"].contiguous()
    for name in ("q_weight", "k_weight"):
        st[name] = (1.0 - case["offset"] + 0.3 * torch.randn(d, device="cuda", generator=gen)).to(_DT[case["weight"]])
    angle = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * torch.from_numpy(_inv_freq(case["rot"])).cuda()
    st["table"] = torch.stack([torch.cos(angle), torch.sin(angle)], -1).float()  # [positions, rot / 2, 2]
    if op == "qk":
        st["positions"] = torch.randint(0, POSITIONS, (rows,), device="cuda", generator=gen).int()
        return st
    st["positions"] = torch.cat([torch.arange(l, l + n) for n, l in zip(news, lens)]).int().cuda()
    p = case["page"]
    need = [-(-(n + l) // p) for n, l in zip(news, lens)]
    pages = sum(need) + 1
    order = torch.from_numpy(np.random.default_rng(seed).permutation(pages)).cuda()
    pt = torch.full((len(news), max(need)), -1, dtype=torch.int32, device="cuda")
    for b, (at, k) in enumerate(zip(_starts(need), need)):
        pt[b, :k] = order[at:at + k]
    slots = pages * p * kv
    st["cache"] = dict(k=torch.zeros(slots * (d + d // 32 * 2), dtype=torch.uint8, device="cuda"), pages=pages, table=pt,
                       v=torch.zeros(slots * (d * (8 if case["v"] == "q8" else 4) // 8 + 2), dtype=torch.uint8, device="cuda"))
    st.update(news=news, lens=lens, starts=_i32(_starts(news)), lengths=_i32(lens))
    return st


# ------------------------------------------------------------------ the framework's calls
_ctx = None


def _own(st):
    global _ctx
    import dyninfer_amd as d
    if _ctx is None:
        _ctx = d.Context(torch.cuda.current_device())
    c = st["case"]
    if c["op"] == "logprobs":
        return tuple(_ctx.token_logprobs(st["logits"], st["tokens"], top=c["top"], temperature=st["temperature"]))
    if c["op"] == "attend":
        rows = st["q"].shape[0]
        lse = torch.empty((rows, c["q_heads"]), dtype=torch.float32, device="cuda")
        batch = d.PromptBatch(st["starts"], max(st["news"]), st["key_starts"], max(n + l for n, l in zip(st["news"], st["lens"])))
        return _ctx.prompt_attention(st["q"], st["k"], st["v"], batch, scale=st["scale"], lse=lse), lse
    rope = d.Rope(st["table"], st["positions"], c["rot"], c["layout"])
    norms = dict(q_norm=d.HeadNorm(st["q_weight"], EPS, c["offset"]), k_norm=d.HeadNorm(st["k_weight"], EPS, c["offset"]))
    if c["op"] == "qk":
        return _ctx.qk_norm_rope(st["q"], st["k"], rope, **norms)
    cc = st["cache"]
    cache = d.KVCache(cc["k"], cc["v"], cc["pages"], c["kv_heads"], c["dim"], c["page"], d.KV_Q8,
                      d.KV_Q8 if c["v"] == "q8" else d.KV_Q4)
    batch = d.KVBatch(cc["table"], st["lengths"], st["starts"], sum(st["news"]), max(st["news"]),
                      max(n + l for n, l in zip(st["news"], st["lens"])))
    q = _ctx.kv_append(cache, batch, st["k"], st["v"], rope=rope, q=st["q"], **norms)
    return (q, *_ctx.kv_read(cache, batch, dtype=torch.bfloat16))


# ------------------------------------------------------------------ the plain forms
def _norm_rope(x, weight, st):
    """f32 x [tokens, heads, d]: each head over its root mean square, times the weight, the first ``rot`` dims rotated."""
    c = st["case"]
    r = c["rot"]
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (weight.float() + c["offset"])
    t = st["table"][st["positions"].long()][:, None]
    cos, sin = t[..., 0], t[..., 1]
    z = y.clone()
    if c["layout"] == "half":
        a, b = y[..., :r // 2], y[..., r // 2:r]
        z[..., :r // 2], z[..., r // 2:r] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        z[..., 0:r:2], z[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    return z


def _stored(x, bits, group):
    """What the codes of f32 x in groups of ``group`` along its last axis stand for."""
    g = x.unflatten(-1, (-1, group))
    top, low = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    s = torch.maximum(top, -low) / 127.0 if bits == 8 else torch.where(top > -low, top, low) / -8.0
    s = s.bfloat16().float()
    y = torch.where(s == 0, torch.zeros_like(g), torch.round(g / s))
    return ((y.clamp(-127, 127) if bits == 8 else y.clamp(-8, 7)) * s).flatten(-2)


def _plain_attend(st):
    c = st["case"]
    kv, d = c["kv_heads"], c["dim"]
    g = c["q_heads"] // kv
    outs, lses, at, from_ = [], [], 0, 0
    for n, l in zip(st["news"], st["lens"]):
        see = torch.arange(n + l, device="cuda")[None] <= torch.arange(l, l + n, device="cuda")[:, None]
        o = torch.empty((kv, n, g, d), device="cuda")
        z = torch.empty((kv, n, g), device="cuda")
        for h in range(kv):  # one head at a time: the scores of all would not fit beside three states
            k, v = (st[x][from_:from_ + n + l, h].float().contiguous() for x in ("k", "v"))
            q = st["q"][at:at + n, h * g:(h + 1) * g].float().reshape(n * g, d)
            s = ((q @ k.t().contiguous()) * st["scale"]).view(n, g, n + l)
            s.masked_fill_(~see[:, None], float("-inf"))
            m = s.amax(-1, keepdim=True)
            e = torch.exp(s - m)
            t = e.sum(-1, keepdim=True)
            o[h] = ((e.view(n * g, n + l) @ v).view(n, g, d)) / t
            z[h] = (m + torch.log(t))[..., 0]
        outs.append(o.permute(1, 0, 2, 3).reshape(n, c["q_heads"], d))
        lses.append(z.permute(1, 0, 2).reshape(n, c["q_heads"]))
        at, from_ = at + n, from_ + n + l
    return torch.cat(outs).to(_DT[c["io"]]), torch.cat(lses)


def _plain_logprobs(st):
    c, tokens = st["case"], st["tokens"]
    x = st["logits"].float()
    vocab = torch.arange(x.shape[1], device="cuda")
    m = x.amax(-1, keepdim=True)
    first = torch.where(x == m, vocab, x.shape[1]).amin(-1, keepdim=True)
    t = torch.ones_like(m) if st["temperature"] is None else st["temperature"][:, None]
    y = (x - m) / torch.where(t > 0, t, torch.ones_like(t))
    y = torch.where(t > 0, y, torch.where(vocab == first, 0.0, float("-inf")))
    e = torch.exp(y)
    z = e.sum(-1, keepdim=True)
    logp = y - torch.log(z)
    entropy = -torch.where(e > 0, e / z * logp, 0.0).sum(-1)
    xt = x.gather(1, tokens[:, None])
    rank = ((x > xt) | ((x == xt) & (vocab < tokens[:, None]))).sum(-1).int()
    chosen = logp.gather(1, tokens[:, None])[:, 0]
    if not c["top"]:
        return chosen, rank, entropy
    bits = (x + 0.0).view(torch.int32)  # as whole numbers of the same order, ties by the lower token
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + ((1 << 32) - 1 - vocab)
    best = (1 << 32) - 1 - (key.topk(c["top"], -1).values & ((1 << 32) - 1))
    there = x.gather(1, best) > float("-inf")
    return chosen, rank, entropy, torch.where(there, best, -1), torch.where(there, logp.gather(1, best), float("-inf"))


def _plain(st):
    c = st["case"]
    if c["op"] == "logprobs":
        return _plain_logprobs(st)
    if c["op"] == "attend":
        return _plain_attend(st)
    q, k = (_norm_rope(st[x].float(), st[x + "_weight"], st) for x in ("q", "k"))
    if c["op"] == "qk":
        return q.to(_DT[c["io"]]), k.to(_DT[c["io"]])
    v = _stored(st["v"].float(), 8 if c["v"] == "q8" else 4, c["dim"])
    return q.to(_DT[c["io"]]), _stored(k, 8, 32).bfloat16(), v.bfloat16()


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ in 64 bits, from the definitions
def _exact_norm_rope(x, weight, st):
    c = st["case"]
    r = c["rot"]
    x = x.double()
    x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * (weight.double() + c["offset"])
    a = st["positions"].double()[:, None] * torch.from_numpy(_inv_freq(r)).cuda()
    z = torch.polar(torch.ones_like(a), a)[:, None]
    head = x[..., :r]
    if c["layout"] == "half":
        w = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * z
        turned = torch.cat([w.real, w.imag], -1)
    else:
        turned = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _exact_stored(x, bits, group):
    shape = x.shape
    x = x.reshape(-1, group)
    hi, lo = x.amax(1), x.amin(1)
    scale = torch.maximum(hi.abs(), lo.abs()) / 127 if bits == 8 else -torch.where(hi > -lo, hi, lo) / 8
    scale = scale.float().bfloat16().double()
    codes = (x / scale[:, None]).nan_to_num(0.0).round()
    lim = (-127, 127) if bits == 8 else (-8, 7)
    return (codes.clamp(*lim) * scale[:, None]).reshape(shape)


def _exact_attend(st):
    c = st["case"]
    g = c["q_heads"] // c["kv_heads"]
    rows = st["q"].shape[0]
    out = torch.zeros((rows, c["q_heads"], c["dim"]), dtype=torch.float64, device="cuda")
    lse = torch.zeros((rows, c["q_heads"]), dtype=torch.float64, device="cuda")
    at, from_ = 0, 0
    for n, l in zip(st["news"], st["lens"]):
        hidden = torch.ones((n, n + l), dtype=torch.bool, device="cuda").triu(l + 1)
        for h in range(c["q_heads"]):
            k, v = (st[x][from_:from_ + n + l, h // g].double().contiguous() for x in ("k", "v"))
            s = (st["q"][at:at + n, h].double() @ k.T.contiguous()) * st["scale"]
            s[hidden] = float("-inf")
            lse[at:at + n, h] = torch.logsumexp(s, -1)
            out[at:at + n, h] = torch.softmax(s, -1) @ v
        at, from_ = at + n, from_ + n + l
    return out, lse


def _exact_logprobs(st):
    c = st["case"]
    got = []
    for b in range(c["rows"]):
        x, tok = st["logits"][b].double(), int(st["tokens"][b])
        order = torch.sort(x, descending=True, stable=True).indices
        t = 1.0 if st["temperature"] is None else float(st["temperature"][b])
        if t > 0:
            logp = torch.log_softmax(x / t, 0)
        else:
            logp = torch.full_like(x, float("-inf"))
            logp[order[0]] = 0.0
        p = logp.exp()
        best = order[:c["top"]]
        there = x[best] > float("-inf")
        got.append((logp[tok], (order == tok).nonzero()[0, 0].int(), -torch.special.xlogy(p, p).sum(),
                    torch.where(there, best, -1), torch.where(there, logp[best], float("-inf"))))
    return tuple(torch.stack(x) for x in zip(*got))[:5 if c["top"] else 3]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(st)
    if case["op"] == "attend":
        return _exact_attend(st)
    q, k = (_exact_norm_rope(st[x], st[x + "_weight"], st) for x in ("q", "k"))
    if case["op"] == "qk":
        return q, k
    return q, _exact_stored(k, 8, 32), _exact_stored(st["v"].double(), 8 if case["v"] == "q8" else 4, case["dim"])
