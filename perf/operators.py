"""The operators of a speculative decoding round over a quantised cache, and how their speed is measured.

A serving program drafts a tree of tokens for each sequence, runs the model over all of them at
once, keeps the path the target model agrees with, and goes on.  Besides the linears, one round
needs of every layer: rotary positions, the new keys and values quantised into the paged cache,
attention of the drafted tokens over the cache; and once at the end the verification of the
drafts and the removal of the rejected rows from the cache.  Prompts take the same calls with one
long chain of tokens, and read the cache back where a prefix is shared.

Cases name the operator in ``op``.  Rows of a call are tokens packed sequence after sequence:
row ``starts[b] + i`` is the token at position ``lengths[b] + i`` of sequence b.

The cache's bytes (``_pack_k``, ``_pack_v``): pages of P tokens; the codes of all pages, then the
bf16 scales of all pages.  K codes lie [page, head, token, dims] with a scale for each block of
32 dims, V codes [page, head, 16 tokens, dims, token] with a scale for each token and head.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False  # False: the plain forms; True: the framework's kernels

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_BITS = {"q8": 8, "q4": 4}
VOCAB = 151936


def listed():
    return [
        # The queries of one token of a small model: a call that is all latency.
        dict(name="rope_1token", op="rope", tokens=1, heads=16, dim=128, rot=128, layout="half", scaling="none",
             io="bf16", fused=False),
        # A prompt's queries and keys as slices of one fused projection; a quarter of the head is left unrotated.
        dict(name="rope_prompt_4099", op="rope", tokens=4099, heads=40, dim=128, rot=96, layout="interleaved",
             scaling="linear", io="f32", fused=True),
        # One sequence, one new token (8B heads): rotate, quantise, write, read back.
        dict(name="append_1token", op="append", seqs=1, new=1, ragged=0, length=1000, q_heads=32, kv_heads=8,
             dim=128, rot=128, layout="half", scaling="none", k="q8", v="q8", page=64, io="bf16", commit=False),
        # Sixteen sequences' drafted trees, written, the accepted paths kept, and those rows read back.
        dict(name="append_commit_16x24", op="append", seqs=16, new=24, ragged=1, length=3000, q_heads=16, kv_heads=8,
             dim=64, rot=32, layout="interleaved", scaling="bands", k="q4", v="q4", page=16, io="f32", commit=True),
        # Four prompts of some two thousand tokens written into a long-context cache.
        dict(name="append_prompts_4x2048", op="append", seqs=4, new=2048, ragged=1, length=777, q_heads=32,
             kv_heads=8, dim=128, rot=128, layout="half", scaling="yarn", k="q8", v="q4", page=128, io="bf16",
             commit=False),
        # A short shared prefix read back in f32.
        dict(name="read_517", op="read", seqs=1, new=517, ragged=0, length=0, kv_heads=5, dim=96, k="q4", v="q8",
             page=16, io="f32"),
        # Long prefixes of eight sequences read back for a prefill in bf16.
        dict(name="read_8x16k", op="read", seqs=8, new=16384, ragged=1, length=0, kv_heads=8, dim=128, k="q8", v="q8",
             page=64, io="bf16"),
        # One sequence, one token, a short context of the small model: the smallest attention call.
        dict(name="attend_1x1_701", op="attend", seqs=1, new=1, ragged=0, length=700, q_heads=16, kv_heads=8,
             dim=128, k="q8", v="q8", page=64, io="f32", tree=False, holes=False),
        # Thirty-two sequences with trees of up to eight drafted tokens, contexts of up to 4096: an ordinary step.
        dict(name="attend_32x8_4k", op="attend", seqs=32, new=8, ragged=1, length=4096, q_heads=32, kv_heads=8,
             dim=128, k="q8", v="q8", page=64, io="bf16", tree=True, holes=False),
        # One long document and a wide tree.
        dict(name="attend_1x64_131k", op="attend", seqs=1, new=64, ragged=0, length=131007, q_heads=32, kv_heads=8,
             dim=128, k="q8", v="q4", page=128, io="bf16", tree=True, holes=False),
        # One sequence's chain of four drafts with the draft model's probabilities.
        dict(name="verify_1x5", op="verify", seqs=1, new=5, ragged=0, vocab=VOCAB, probs="f32", io="bf16",
             tree=False),
        # Thirty-two trees of up to 16 nodes drafted without probabilities.
        dict(name="verify_32x16", op="verify", seqs=32, new=16, ragged=1, vocab=VOCAB, probs="", io="f32", tree=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "append", "read", "attend", "attend", "attend", "verify", "verify"])
    io = rng.choice(["f32", "bf16"])
    if op == "verify":
        c = dict(op=op, seqs=_log(rng, 1, 32), new=_log(rng, 1, 16), ragged=rng.choice([0, rng.randint(1, 10**6)]),
                 vocab=rng.choice([VOCAB, _log(rng, 1000, VOCAB)]), probs=rng.choice(["", "f32", "bf16"]), io=io,
                 tree=rng.random() < 0.5)
        if c["probs"]:
            c["seqs"] = max(1, c["seqs"] // 2)
        return c
    dim = rng.choice([64, 96, 128, 128, 256])
    heads = dict(dim=dim, kv_heads=_log(rng, 1, 16))
    turn = dict(rot=rng.choice([dim, dim, dim // 2, 24]), layout=rng.choice(["half", "interleaved"]),
                scaling=rng.choice(["none", "linear", "yarn", "bands"]))
    if op == "rope":
        c = dict(op=op, tokens=_log(rng, 1, 4099), heads=_log(rng, 1, 64), dim=dim, io=io, fused=rng.random() < 0.5, **turn)
        c["tokens"] = max(1, min(c["tokens"], 4099 * 40 * 128 // (c["heads"] * dim)))
        return c
    store = dict(k=rng.choice(["q8", "q8", "q4"]), v=rng.choice(["q8", "q4"]), page=rng.choice([16, 32, 64, 128, 256]),
                 seqs=_log(rng, 1, 64), ragged=rng.choice([0, rng.randint(1, 10**6), rng.randint(1, 10**6)]))
    if op == "append":
        c = dict(op=op, new=_log(rng, 1, 4096), length=_log(rng, 1, 16384), io=io, commit=rng.random() < 0.4,
                 q_heads=heads["kv_heads"] * rng.choice([1, 2, 3, 4, 8]), **heads, **turn, **store)
        if c["commit"]:
            c["new"] = min(c["new"], 64)
        c["new"] = max(1, min(c["new"], 8192 * 48 * 128 // (c["seqs"] * (c["q_heads"] + 2 * c["kv_heads"]) * dim)))
        return c
    if op == "read":
        c = dict(op=op, new=_log(rng, 1, 65536), length=rng.choice([0, 0, _log(rng, 1, 3000)]), io=io, **heads, **store)
        c["new"] = max(1, min(c["new"], 8 * 16384 * 8 * 128 // (c["seqs"] * c["kv_heads"] * dim * (2 if io == "f32" else 1))))
        return c
    c = dict(op=op, new=_log(rng, 1, 64), length=_log(rng, 1, 131007), io=io, tree=rng.random() < 0.7,
             holes=rng.random() < 0.3, q_heads=heads["kv_heads"] * rng.choice([1, 2, 3, 4, 4, 8]), **heads, **store)
    c["seqs"] = min(c["seqs"], max(1, 64 * 131071 * 32 * 128 // (c["new"] * (c["length"] + c["new"]) * c["q_heads"] * dim)))
    c["seqs"] = min(c["seqs"], max(1, 131071 * 8 * 128 // ((c["length"] + c["new"]) * c["kv_heads"] * dim)))
    most = 64 * 131071 * 32 * 128 // (c["new"] * c["seqs"] * c["q_heads"] * dim)
    c["length"] = max(1, min(c["length"], most, 131071 * 8 * 128 // (c["kv_heads"] * dim)) - c["new"])
    return c


# ------------------------------------------------------------------ what a case's sizes are
def _sizes(case):
    """New tokens and committed lengths of each sequence; where they differ, ``ragged`` numbers their choice."""
    rng = random.Random(case["ragged"])
    n, new = case["seqs"], case["new"]
    news = [rng.randint((new + 1) // 2, new) if case["ragged"] else new for _ in range(n)]
    news[rng.randrange(n)] = new
    top = case.get("length", 0)
    if case["ragged"] and top:
        lens = [rng.randint(top // 4, top) for _ in range(n)]
        lens[rng.randrange(n)] = top
        if n > 3:
            lens[rng.randrange(n)] = 0  # a sequence that has only just begun
    else:
        lens = [top] * n
    return news, lens


def _row_bytes(case):
    """Bytes of one token's K and V of all kv heads in the cache."""
    d = case["dim"]
    return case["kv_heads"] * (d * _BITS[case["k"]] / 8 + d // 32 * 2 + d * _BITS[case["v"]] / 8 + 2)


def work(case):
    op, e = case["op"], 4 if case["io"] == "f32" else 2
    if op == "rope":
        t, h, d, r = case["tokens"], case["heads"], case["dim"], case["rot"]
        return {"bytes": t * (2 * h * d * e + r * 4 + 4), "flops": 3 * t * h * r}
    if op == "verify":
        rows = sum(_sizes(case)[0])
        n, v = case["seqs"], case["vocab"]
        b = rows * v * e + n * v * 4  # every logit once, the noise of the one draw a sequence
        f = rows * v * 4 + n * v * 2
        if case["probs"]:
            b += n * v * (4 if case["probs"] == "f32" else 2)
            f += n * v * 2
        return {"bytes": int(b), "flops": int(f)}
    news, lens = _sizes(case)
    new, d, kv = sum(news), case["dim"], case["kv_heads"]
    row = _row_bytes(case)
    if op == "read":
        return {"bytes": int(new * (row + 2 * kv * d * e)), "flops": int(new * kv * d * 2)}
    if op == "append":
        q = case["q_heads"]
        # q, k, v in; q out; the codes written; those kept read again, their values written
        kept = sum(len(p) for p in _paths(case)) if case["commit"] else new
        return {"bytes": int(new * ((2 * q + 2 * kv) * d * e + case["rot"] * 4 + row) + kept * (row + 2 * kv * d * e)),
                "flops": int(new * (3 * (q + kv) * case["rot"] + 6 * kv * d))}
    return {"bytes": int((sum(lens) + new) * row + 2 * new * case["q_heads"] * d * e),
            "flops": sum(4 * n * case["q_heads"] * d * (l + n) for n, l in zip(news, lens))}


# ------------------------------------------------------------------ rotary tables
def _inv_freq(case):
    """Angle per position of each pair, in 64 bits, and the factor on cosine and sine."""
    r, theta, factor, orig = case["rot"], 1.0e6 if case["scaling"] == "none" else 1.0e4, 8.0, 4096.0
    i = np.arange(r // 2, dtype=np.float64)
    f = theta ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        turn = lambda beta: r * math.log(orig / (beta * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), r - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if case["scaling"] == "bands":
        wave, low, high = 2 * math.pi / f, 1.0, 4.0
        s = np.clip((orig / wave - low) / (high - low), 0, 1)
        return (1 - s) * f / factor + s * f, 1.0
    return f, 1.0


def _table(case, positions):
    f, m = _inv_freq(case)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * torch.from_numpy(f).cuda()
    return torch.stack([torch.cos(a) * m, torch.sin(a) * m], -1).float()  # [positions, rot/2, 2]


# ------------------------------------------------------------------ the cache's codes and bytes
def _quant(x, bits, group):
    """Codes and scales of f32 x [..., n] in groups of ``group`` along the last axis."""
    g = x.unflatten(-1, (-1, group))
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    g = torch.where(bad, torch.zeros_like(g), g)
    top, low = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    if bits == 8:
        s = (torch.maximum(top, -low) / 127.0).bfloat16().float()
    else:
        s = (torch.where(top > -low, top, low) / -8.0).bfloat16().float()
    c = torch.where(s == 0, torch.zeros_like(g), torch.round(g / s))
    c = c.clamp(-127, 127) if bits == 8 else c.clamp(-8, 7)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    return c.flatten(-2), s.squeeze(-1)


def _k_order(d):
    """The dim at each place of a K row: pairs of 32-blocks lie [4 parts of 8 dims][block of the pair]."""
    out = []
    for b in range(0, d // 32, 2):
        pair = [x for x in (b, b + 1) if x < d // 32]
        out += [32 * x + 8 * part + j for part in range(4) for x in pair for j in range(8)]
    return out


def _nibbles(u):
    """[..., 8n] codes 0..15 -> [..., 4n] bytes: byte t of a group of eight holds codes t and t + 4."""
    u = u.unflatten(-1, (-1, 2, 4))
    return (u[..., 0, :] | (u[..., 1, :] << 4)).flatten(-2)


def _un_nibbles(b):
    b = b.unflatten(-1, (-1, 1, 4))
    return torch.cat([b & 15, b >> 4], -2).flatten(-3)


def _pack_k(codes, scales, bits, page):
    """codes [slots, heads, d], scales [slots, heads, d/32] -> the K buffer."""
    n, h, d = codes.shape
    u = (codes.to(torch.int32) + (128 if bits == 8 else 8)).to(torch.uint8)[..., torch.tensor(_k_order(d), device=codes.device)]
    u = u if bits == 8 else _nibbles(u)
    u = u.unflatten(0, (-1, page)).transpose(1, 2).contiguous()
    s = scales.bfloat16().unflatten(0, (-1, page)).transpose(1, 2).contiguous()
    return torch.cat([u.flatten(), s.flatten().view(torch.uint8)])


def _pack_v(codes, scales, bits, page):
    """codes [slots, heads, d], scales [slots, heads] -> the V buffer."""
    u = codes.to(torch.int32).unflatten(0, (-1, page // 16, 16)).permute(0, 3, 1, 4, 2)  # page, head, chunk, dim, token
    u = (u & 255).to(torch.uint8) if bits == 8 else _nibbles((u & 15).to(torch.uint8))
    s = scales.bfloat16().unflatten(0, (-1, page)).transpose(1, 2).contiguous()
    return torch.cat([u.contiguous().flatten(), s.flatten().view(torch.uint8)])


def _unpack(buf, kind, bits, pages, page, heads, d, want):
    """Values [tokens, heads, d] in f32 of the pages ``want`` (a tensor) of a K or V buffer."""
    nc = pages * heads * page * d * bits // 8
    if kind == "k":
        u = buf[:nc].view(pages, heads, page, d * bits // 8)[want]
        u = (u if bits == 8 else _un_nibbles(u)).float() - (128 if bits == 8 else 8)
        back = torch.empty(d, dtype=torch.int64)
        back[torch.tensor(_k_order(d))] = torch.arange(d)
        u = u[..., back.to(buf.device)]
        s = buf[nc:].view(torch.bfloat16).view(pages, heads, page, d // 32)[want].float()
        x = (u.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)
    else:
        u = buf[:nc].view(pages, heads, page // 16, d, 16 * bits // 8)[want]
        u = u.view(torch.int8).float() if bits == 8 else ((_un_nibbles(u).to(torch.int32) ^ 8) - 8).float()
        u = u.transpose(-1, -2).flatten(2, 3)
        x = u * buf[nc:].view(torch.bfloat16).view(pages, heads, page)[want].float()[..., None]
    return x.transpose(1, 2).flatten(0, 1)


# ------------------------------------------------------------------ inputs
def _kv(gen, n, heads, d, key):
    """Keys (a few strong channels, as rotary keys have) or values in f32."""
    x = torch.randn((n, heads, d), device="cuda", generator=gen)
    if key:
        x *= torch.where(torch.rand((1, heads, d), device="cuda", generator=gen) < 0.05, 6.0, 1.0)
    else:
        x *= 0.3 + torch.rand((n, heads, 1), device="cuda", generator=gen)
    return x


def _cache(case, seed, tokens, gen, filled):
    """A cache with room for ``tokens`` of each sequence on shuffled pages, its page table."""
    p, kv, d = case["page"], case["kv_heads"], case["dim"]
    need = [max(1, -(-t // p)) for t in tokens]
    pages, width = sum(need) + 1, max(need)
    order = torch.from_numpy(np.random.default_rng(seed).permutation(pages)).cuda()
    table = torch.full((len(tokens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    kb, vb = _BITS[case["k"]], _BITS[case["v"]]
    if filled:
        kc, ks = _quant(_kv(gen, pages * p, kv, d, True), kb, 32)
        k = _pack_k(kc, ks, kb, p)
        vc, vs = _quant(_kv(gen, pages * p, kv, d, False), vb, d)
        v = _pack_v(vc, vs[..., 0], vb, p)
    else:
        k = torch.zeros(pages * p * kv * (d * kb // 8 + d // 32 * 2), dtype=torch.uint8, device="cuda")
        v = torch.zeros(pages * p * kv * (d * vb // 8 + 2), dtype=torch.uint8, device="cuda")
    return dict(k=k, v=v, pages=pages, table=table, need=need)


def _trees(case, news, seed):
    """Parents of every node of every sequence's tree (a chain where the case says so)."""
    rng = random.Random(7919 * seed + 3)
    return [[-1] + [rng.randint(max(0, i - 4), i - 1) if case["tree"] else i - 1 for i in range(1, n)] for n in news]


def _paths(case):
    """The path of each sequence's tree that is kept: a node and its ancestors."""
    news, rng, paths = _sizes(case)[0], random.Random(case["ragged"] + 5), []
    for t in _trees(dict(tree=True), news, case["ragged"]):
        node, path = rng.randrange(len(t)), []
        while node >= 0:
            path.append(node)
            node = t[node]
        paths.append(path[::-1])
    return paths


def _starts(news):
    return [0] + np.cumsum(news).tolist()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2654435761 % (1 << 62))
    op, dt = case["op"], _DT[case["io"]]
    st = dict(case=case)
    if op == "rope":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        wide = torch.randn((t, h + 8, d), device="cuda", generator=gen).to(dt)
        st["x"] = wide[:, :h] if case["fused"] else wide[:, :h].contiguous()
        st["table"] = _table(case, 32768)
        st["positions"] = torch.randint(0, 32768, (t,), device="cuda", generator=gen).int()
    elif op == "verify":
        news, _ = _sizes(case)
        rows, v = sum(news), case["vocab"]
        trees = _trees(case, news, seed)
        starts = _starts(news)
        logits = torch.randn((rows, v), device="cuda", generator=gen) * 2.5
        logits += 6.0 * (torch.rand((rows, v), device="cuda", generator=gen) < 8.0 / v)  # a few likely tokens
        logits = logits.to(dt)
        near = logits.float() + 0.5 * torch.randn((rows, v), device="cuda", generator=gen)
        probs = torch.softmax(near, -1)
        parent_rows = [starts[b] + max(p, 0) for b, t in enumerate(trees) for p in t]
        if case["probs"]:
            src = probs[torch.tensor(parent_rows, device="cuda")]
            tokens = torch.multinomial(src, 1, generator=gen)[:, 0]
        else:  # the draft's most likely tokens, the next sibling takes the next one
            rank = [sum(1 for q in t[1:i] if q == t[i]) if i else 0 for t in trees for i in range(len(t))]
            best = near.topk(max(rank) + 1, -1).indices
            tokens = best[torch.tensor(parent_rows, device="cuda"), torch.tensor(rank, device="cuda")]
        temp = torch.rand(len(news), device="cuda", generator=gen) * 0.6 + 0.7
        temp[torch.rand(len(news), device="cuda", generator=gen) < 0.2] = 0.0  # some sequences decode greedily
        st.update(news=news, trees=trees, starts=_i32(starts), logits=logits, tokens=tokens.contiguous(),
                  parents=_i32([p for t in trees for p in t]), temperature=temp,
                  probs=probs.to(_DT[case["probs"]]) if case["probs"] else None,
                  uniform=torch.rand(rows, device="cuda", generator=gen),
                  noise=torch.empty((len(news), v), device="cuda").exponential_(generator=gen).clamp_min_(1e-30))
    else:
        news, lens = _sizes(case)
        st.update(news=news, lens=lens, starts=_i32(_starts(news)), lengths=_i32(lens),
                  cache=_cache(case, seed, [a + b for a, b in zip(news, lens)], gen, op != "append"))
        rows, d, kv = sum(news), case["dim"], case["kv_heads"]
        if op == "append":
            qkv = torch.cat([torch.randn((rows, case["q_heads"], d), device="cuda", generator=gen),
                             _kv(gen, rows, kv, d, True), _kv(gen, rows, kv, d, False)], 1).to(dt)
            st["q"], st["k"], st["v"] = qkv[:, :case["q_heads"]], qkv[:, -2 * kv:-kv], qkv[:, -kv:]
            st["table"] = _table(case, max(a + b for a, b in zip(news, lens)) + 1)
            if case["commit"]:  # positions go by depth in the tree, and a path of each tree is kept
                pos, paths, width = [], _paths(case), max(news)
                for t, n0 in zip(_trees(dict(tree=True), news, case["ragged"]), lens):
                    depth = [0] * len(t)
                    for i in range(1, len(t)):
                        depth[i] = depth[t[i]] + 1
                    pos += [n0 + x for x in depth]
                st.update(paths=paths, path=_i32([p + [-1] * (width - len(p)) for p in paths]),
                          counts=_i32([len(p) for p in paths]), kept=_i32(_starts([len(p) for p in paths])))
                st["positions"] = _i32(pos)
            else:
                st["positions"] = torch.cat([torch.arange(l, l + n) for n, l in zip(news, lens)]).int().cuda()
        elif op == "attend":
            st["q"] = torch.randn((rows, case["q_heads"], d), device="cuda", generator=gen).to(dt)
            st["scale"] = d ** -0.5
            st["mask"] = None
            if case["tree"]:
                rng = random.Random(seed + 11)
                bits = []
                for t in _trees(case, news, seed):
                    seen = []
                    for i, p in enumerate(t):
                        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
                    if case["holes"]:  # rows that see no drafted token, the padding of a batch
                        seen = [0 if rng.random() < 0.2 else s for s in seen]
                    bits += [s - (1 << 64) if s >> 63 else s for s in seen]
                st["mask"] = torch.tensor(bits, dtype=torch.int64, device="cuda")[:, None]
    return st


# ------------------------------------------------------------------ the framework's calls
_ctx = None


def _own(st):
    global _ctx
    import dyninfer_amd as d
    if _ctx is None:
        _ctx = d.Context(torch.cuda.current_device())
    c = st["case"]
    op = c["op"]
    if op == "rope":
        return _ctx.rope(st["x"], d.Rope(st["table"], st["positions"], c["rot"], c["layout"]))
    if op == "verify":
        return _ctx.draft_verify(st["logits"], st["tokens"], st["parents"], st["starts"], max(st["news"]),
                                 draft_probs=st["probs"], temperature=st["temperature"], uniform=st["uniform"],
                                 noise=st["noise"])
    enc = {"q8": d.KV_Q8, "q4": d.KV_Q4}
    cc = st["cache"]
    cache = d.KVCache(cc["k"], cc["v"], cc["pages"], c["kv_heads"], c["dim"], c["page"], enc[c["k"]], enc[c["v"]])
    batch = d.KVBatch(cc["table"], st["lengths"], st["starts"], sum(st["news"]), max(st["news"]),
                      max(st["lens"]) + max(st["news"]))
    if op == "read":
        return _ctx.kv_read(cache, batch, dtype=_DT[c["io"]])
    if op == "attend":
        return _ctx.tree_attention(cache, batch, st["q"], mask=st["mask"], scale=st["scale"])
    q = _ctx.kv_append(cache, batch, st["k"], st["v"], q=st["q"],
                       rope=d.Rope(st["table"], st["positions"], c["rot"], c["layout"]))
    if c["commit"]:
        _ctx.kv_commit(cache, batch, st["path"], st["counts"])
        n = [len(p) for p in st["paths"]]
        batch = d.KVBatch(cc["table"], st["lengths"], st["kept"], sum(n), max(n), max(st["lens"]) + max(n))
    return (q, *_ctx.kv_read(cache, batch, dtype=_DT[c["io"]]))


# ------------------------------------------------------------------ the plain forms
def _rotate(x, table, positions, rot, layout):
    """f32 x [tokens, heads, d] with its first ``rot`` dims rotated."""
    t = table[positions.long()][:, None]
    c, s = t[..., 0], t[..., 1]
    y = x.clone()
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    return y


def _values(st, kind, b, first, count):
    """f32 values of positions first..first+count of sequence b."""
    c, cc = st["case"], st["cache"]
    p0, p1 = first // c["page"], -(-(first + count) // c["page"])
    want = cc["table"][b, p0:p1].long()
    x = _unpack(cc[kind], kind, _BITS[c[kind]], cc["pages"], c["page"], c["kv_heads"], c["dim"], want)
    return x[first - p0 * c["page"]:][:count]


def _plain_attend(st):
    c = st["case"]
    kv, d = c["kv_heads"], c["dim"]
    g = c["q_heads"] // kv
    outs, at = [], 0
    for b, (n, l) in enumerate(zip(st["news"], st["lens"])):
        k, v = _values(st, "k", b, 0, l + n), _values(st, "v", b, 0, l + n)
        q = st["q"][at:at + n].float().view(n, kv, g, d).permute(1, 0, 2, 3).reshape(kv, n * g, d)
        s = torch.bmm(q, k.permute(1, 2, 0).contiguous()) * st["scale"]
        j = torch.arange(n, device=s.device)
        if st["mask"] is None:
            see = j[None, :] <= j[:, None]
        else:
            see = (st["mask"][at:at + n] >> j[None, :]) & 1 != 0
        see = see.repeat_interleave(g, 0)
        s[:, :, l:] = torch.where(see, s[:, :, l:], torch.full_like(s[:, :, l:], float("-inf")))
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
        e = torch.exp(s - m)
        z = e.sum(-1, keepdim=True)
        o = torch.bmm(e, v.permute(1, 0, 2).contiguous()) / torch.where(z == 0, torch.ones_like(z), z)
        outs.append(o.view(kv, n, g, d).permute(1, 0, 2, 3).reshape(n, c["q_heads"], d))
        at += n
    return torch.cat(outs).to(_DT[c["io"]])


def _plain_verify(st):
    news, dev = st["news"], st["logits"].device
    n, width = len(news), max(news)
    base = st["starts"][:-1].long()
    count = st["starts"][1:].long() - base
    parents, tokens, uniform = st["parents"].long(), st["tokens"].long(), st["uniform"]
    logits, probs, temp = st["logits"], st["probs"], st["temperature"][:, None]
    greedy = temp <= 0
    vocab = torch.arange(logits.shape[1], device=dev)[None]

    def target(rows):
        x = logits[rows].float()
        x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x).clamp_max(torch.finfo(torch.float32).max)
        m = x.amax(-1, keepdim=True)
        first = torch.where(x == m, vocab, logits.shape[1]).amin(-1, keepdim=True)
        e = torch.exp((x - m) / torch.where(greedy, torch.ones_like(temp), temp))
        e = torch.where(greedy, (vocab == first).float(), e / e.sum(-1, keepdim=True))
        return torch.where(m == float("-inf"), torch.zeros_like(e), e)

    cur = torch.zeros(n, dtype=torch.int64, device=dev)
    left = target(base)  # what of the current node's distribution is left to draw from
    full = left
    path = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    counts = torch.ones(n, dtype=torch.int64, device=dev)
    spent = torch.zeros(n, dtype=torch.bool, device=dev)
    lanes = torch.arange(n, device=dev)
    for i in range(1, width):
        row = torch.where(i < count, base + i, base)
        child = (i < count) & (parents[row] == cur) & ~spent
        tok = tokens[row]
        ok = (tok >= 0) & (tok < logits.shape[1])
        tok = torch.where(ok, tok, torch.zeros_like(tok))
        p = torch.where(ok, left[lanes, tok], torch.zeros_like(uniform[row]))
        without = torch.where((vocab == tok[:, None]) & ok[:, None], torch.zeros_like(left), left)
        if probs is None:
            q = torch.ones_like(p)
            rest = without
        else:
            qrow = probs[base + cur].float()
            q = qrow[lanes, tok]
            rest = torch.where(greedy, without, (left - qrow).clamp_min(0.0))
        take = torch.where(greedy[:, 0], p > 0, uniform[row] * q < p)
        yes, no = child & take, child & ~take
        z = rest.sum(-1, keepdim=True)
        spent = torch.where(no & (z[:, 0] <= 0), torch.ones_like(spent), spent)
        rest = torch.where(z > 0, rest / torch.where(z > 0, z, torch.ones_like(z)), full)
        cur = torch.where(yes, torch.full_like(cur, i), cur)
        path = torch.where(yes[:, None] & (torch.arange(width, device=dev)[None] == counts[:, None]), i, path).int()
        counts = counts + yes.long()
        fresh = target(base + cur)
        full = torch.where(yes[:, None], fresh, full)
        left = torch.where(yes[:, None], fresh, torch.where(no[:, None], rest, left))
        spent = spent & ~yes
    score = torch.where(greedy, left, left / st["noise"])
    best = score.amax(-1, keepdim=True)
    token = torch.where(score == best, vocab, logits.shape[1]).amin(-1)
    token = torch.where(best[:, 0] > 0, token, torch.full_like(token, -1))
    return path, counts.int(), token


def _plain(st):
    c = st["case"]
    op = c["op"]
    if op == "rope":
        return _rotate(st["x"].float(), st["table"], st["positions"], c["rot"], c["layout"]).to(_DT[c["io"]])
    if op == "verify":
        return _plain_verify(st)
    if op == "attend":
        return _plain_attend(st)
    if op == "read":
        return tuple(torch.cat([_values(st, kind, b, l, n) for b, (n, l) in enumerate(zip(st["news"], st["lens"]))])
                     .to(_DT[c["io"]]) for kind in ("k", "v"))
    turn = (st["table"], st["positions"], c["rot"], c["layout"])
    q = _rotate(st["q"].float(), *turn).to(_DT[c["io"]])
    kc, ks = _quant(_rotate(st["k"].float(), *turn), _BITS[c["k"]], 32)
    vc, vs = _quant(st["v"].float(), _BITS[c["v"]], c["dim"])
    k = (kc.unflatten(-1, (-1, 32)) * ks[..., None]).flatten(-2)
    v = vc * vs
    if c["commit"]:
        rows, at = [], 0
        for n, p in zip(st["news"], st["paths"]):
            rows += [at + i for i in p]
            at += n
        rows = torch.tensor(rows, device=k.device)
        k, v = k[rows], v[rows]
    return q, k.to(_DT[c["io"]]), v.to(_DT[c["io"]])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ in 64 bits, from the definitions
def _exact_codes(x, bits, group):
    shape = x.shape
    x = x.reshape(-1, group)
    ends = torch.stack([x.amax(1), x.amin(1)], 1)
    if bits == 8:
        scale = ends.abs().amax(1) / 127
    else:
        scale = -torch.where(ends[:, 0] > -ends[:, 1], ends[:, 0], ends[:, 1]) / 8
    scale = scale.float().bfloat16().double()
    codes = (x / scale[:, None]).nan_to_num(0.0).round()
    lim = (-127, 127) if bits == 8 else (-8, 7)
    return (codes.clamp(*lim) * scale[:, None]).reshape(shape)


def _exact_turn(x, case, positions):
    f, m = _inv_freq(case)
    a = positions.double()[:, None] * torch.from_numpy(f).cuda()
    z = torch.polar(torch.full_like(a, m), a)[:, None]
    r = case["rot"]
    head = x[..., :r]
    if case["layout"] == "half":
        w = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * z
        turned = torch.cat([w.real, w.imag], -1)
    else:
        turned = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _exact_rows(st, kind, b, first, count):
    """f64 values of positions of sequence b, read byte by byte from the layout's definition."""
    c, cc = st["case"], st["cache"]
    bits, page, heads, d = _BITS[c[kind]], c["page"], c["kv_heads"], c["dim"]
    pos = torch.arange(first, first + count, device="cuda")
    pg, tok = cc["table"][b].long()[pos // page], pos % page
    head, dim = torch.arange(heads, device="cuda")[None, :, None], torch.arange(d, device="cuda")[None, None]
    block = (pg[:, None, None] * heads + head) * page
    t = tok[:, None, None]
    if kind == "k":
        blk, part, j = dim // 32, dim % 32 // 8, dim % 8
        pair = 2 - ((blk // 2 * 2 + 2) * 32 > d).long()  # blocks in this dim's pair
        place = (block + t) * d + blk // 2 * 64 + part * 8 * pair + blk % 2 * 8 + j
        scale = (block + t) * (d // 32) + blk
    else:
        place = (block + t // 16 * 16) * d + dim * 16 + t % 16
        scale = block + t
    total = cc["pages"] * heads * page * d * bits // 8
    if bits == 8:
        raw = cc[kind][place].long()
        code = raw - 128 if kind == "k" else raw - 256 * (raw > 127).long()
    else:
        raw = cc[kind][place // 8 * 4 + place % 4].long() >> (4 * (place % 8 // 4))
        raw = raw % 16
        code = raw - 8 if kind == "k" else raw - 16 * (raw > 7).long()
    return code.double() * cc[kind][total:].view(torch.bfloat16)[scale].double()


def _exact_attend(st):
    c = st["case"]
    kv = c["kv_heads"]
    g = c["q_heads"] // kv
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, l) in enumerate(zip(st["news"], st["lens"])):
        sees = torch.ones((n, l + n), dtype=torch.bool)
        for i in range(n):
            word = (1 << (i + 1)) - 1 if st["mask"] is None else int(st["mask"][at + i, 0])
            sees[i, l:] = torch.tensor([word >> j & 1 == 1 for j in range(n)])
        sees = sees.cuda()
        k, v = _exact_rows(st, "k", b, 0, l + n), _exact_rows(st, "v", b, 0, l + n)
        for h in range(kv):
            for x in range(g):
                s = (st["q"][at:at + n, h * g + x].double() @ k[:, h].T.contiguous()) * st["scale"]
                p = torch.softmax(s.masked_fill(~sees, float("-inf")), -1).nan_to_num(0.0)
                out[at:at + n, h * g + x] = p @ v[:, h]
        at += n
    return out


def _exact_verify(st):
    c = st["case"]
    width = max(st["news"])
    paths, counts, tokens, at = [], [], [], 0
    for b, (n, tree) in enumerate(zip(st["news"], st["trees"])):
        temp = float(st["temperature"][b])

        def target(row):
            x = st["logits"][at + row].double()
            if temp <= 0:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1.0
                return p
            return torch.softmax(x / temp, 0)

        node, path = 0, [0]
        left = target(0)
        while True:
            taken = None
            for i in range(node + 1, n):
                if tree[i] != node:
                    continue
                tok, u = int(st["tokens"][at + i]), float(st["uniform"][at + i])
                if temp <= 0 or st["probs"] is None:
                    q = torch.zeros_like(left)
                    q[tok] = 1.0
                    u = 0.0 if temp <= 0 else u
                    rest = left * (1 - q)
                else:
                    q = st["probs"][at + node].double()
                    rest = (left - q).clamp_min(0)
                if u * float(q[tok]) < float(left[tok]):
                    taken = i
                    break
                if float(rest.sum()) <= 0:
                    left = target(node)
                    break
                left = rest / rest.sum()
            if taken is None:
                break
            node = taken
            path.append(node)
            left = target(node)
        score = left if temp <= 0 else left / st["noise"][b].double()
        tokens.append(int(score.argmax()))
        counts.append(len(path))
        paths.append(path + [-1] * (width - len(path)))
        at += n
    return _i32(paths), _i32(counts), torch.tensor(tokens, dtype=torch.int64, device="cuda")


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return _exact_turn(st["x"].double(), case, st["positions"])
    if op == "verify":
        return _exact_verify(st)
    if op == "attend":
        return _exact_attend(st)
    if op == "read":
        return tuple(torch.cat([_exact_rows(st, kind, b, l, n) for b, (n, l) in enumerate(zip(st["news"], st["lens"]))])
                     for kind in ("k", "v"))
    q = _exact_turn(st["q"].double(), case, st["positions"])
    k = _exact_codes(_exact_turn(st["k"].double(), case, st["positions"]), _BITS[case["k"]], 32)
    v = _exact_codes(st["v"].double(), _BITS[case["v"]], case["dim"])
    if case["commit"]:
        rows, at = [], 0
        for n, p in zip(st["news"], st["paths"]):
            rows += [at + i for i in p]
            at += n
        k, v = k[rows], v[rows]
    return q, k, v
