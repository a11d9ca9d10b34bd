"""Plain restatement, in numpy, of the cache's bytes and of the calls around attention
(include/dyninfer_mi355x.h), for the tests to compare with.  Codes and rotations follow the
same f32 operations as the kernels state; attention and verification are in 64 bits."""
import math

import numpy as np
import torch

F32 = np.float32


def bf16(x):
    """f32 array rounded to bf16, as f32."""
    return torch.from_numpy(np.ascontiguousarray(x, dtype=F32)).bfloat16().float().numpy()


def quant(x, bits, group):
    """(codes int, scales f32) of f32 x [..., n] in groups along the last axis."""
    g = x.astype(F32).reshape(*x.shape[:-1], -1, group)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], F32(0), g)
    top, low = g.max(-1), g.min(-1)
    if bits == 8:
        s = bf16(np.maximum(top, -low) / F32(127))
    else:
        s = bf16(np.where(top > -low, top, low) / F32(-8))
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s[..., None] == 0, F32(0), np.rint(g / s[..., None]))
    lim = (-127, 127) if bits == 8 else (-8, 7)
    c = np.clip(c, *lim).astype(np.int64)
    return c.reshape(x.shape), np.where(bad, F32(np.nan), s)


class RefCache:
    """Codes and scales of every slot, from and to the two byte buffers."""

    def __init__(self, pages, heads, dim, page, kb, vb, rng):
        self.pages, self.heads, self.dim, self.page, self.kb, self.vb = pages, heads, dim, page, kb, vb
        r = lambda bits: (-127, 128) if bits == 8 else (-8, 8)
        self.kc = rng.integers(*r(kb), (pages, heads, page, dim))
        self.vc = rng.integers(*r(vb), (pages, heads, page, dim))
        self.ks = bf16(np.exp(rng.normal(-4, 0.5, (pages, heads, page, dim // 32))))
        self.vs = bf16(np.exp(rng.normal(-4, 0.5, (pages, heads, page))))

    def copy(self):
        c = object.__new__(RefCache)
        c.__dict__ = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in self.__dict__.items()}
        return c

    def k_order(self):
        out = []
        for b in range(0, self.dim // 32, 2):
            pair = [x for x in (b, b + 1) if 32 * x < self.dim]
            for part in range(4):
                for x in pair:
                    out += [32 * x + 8 * part + j for j in range(8)]
        return out

    @staticmethod
    def _nib(u):
        u = u.reshape(*u.shape[:-1], -1, 2, 4)
        return (u[..., 0, :] | u[..., 1, :] << 4).reshape(*u.shape[:-3], -1)

    def buffers(self):
        """(k, v) as uint8 arrays."""
        def as_bf16(s):
            bits = torch.from_numpy(np.ascontiguousarray(s)).bfloat16().view(torch.int16).numpy().view(np.uint16)
            return np.where(np.isnan(s), np.uint16(0x7FC0), bits).view(np.uint8).ravel()

        k = self.kc[..., self.k_order()]
        k = k + 128 if self.kb == 8 else self._nib(k + 8)
        v = self.vc.reshape(self.pages, self.heads, self.page // 16, 16, self.dim).swapaxes(-1, -2)
        v = v & 255 if self.vb == 8 else self._nib(v & 15)
        return (np.concatenate([k.astype(np.uint8).ravel(), as_bf16(self.ks)]),
                np.concatenate([v.astype(np.uint8).ravel(), as_bf16(self.vs)]))

    def row(self, page, slot, kind):
        """f64 values [heads, dim] of a slot."""
        if kind == "k":
            return self.kc[page, :, slot] * np.repeat(self.ks[page, :, slot].astype(np.float64), 32, -1)
        return self.vc[page, :, slot] * self.vs[page, :, slot].astype(np.float64)[:, None]

    def rows(self, table, first, count, kind):
        """f64 [count, heads, dim] of positions first.. of a sequence with page table `table`; NaN where absent."""
        out = np.full((count, self.heads, self.dim), np.nan)
        for i in range(count):
            p = (first + i) // self.page
            if p < len(table) and 0 <= table[p] < self.pages:
                out[i] = self.row(table[p], (first + i) % self.page, kind)
        return out


def rotate(x, table, positions, rot, half):
    """f32 x [tokens, heads, dim]; products and sums rounded one by one."""
    y = x.astype(F32).copy()
    for i, p in enumerate(positions):
        if not 0 <= p < len(table):
            y[i, :, :rot] = np.nan
            continue
        c, s = table[p][:, 0], table[p][:, 1]
        a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
        u, v = x[i][:, a].astype(F32), x[i][:, b].astype(F32)
        y[i][:, a], y[i][:, b] = u * c - v * s, u * s + v * c
    return y


def table(positions, rot, theta=10000.0, scaling="none", factor=1.0, original=0.0, fast=32.0, slow=1.0, attn=0.0,
          low=1.0, high=4.0):
    """The rotary table in 64 bits."""
    i = np.arange(rot // 2)
    f = theta ** (-2.0 * i / rot)
    m = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        at = lambda beta: rot * math.log(original / (beta * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        m = attn if attn > 0 else 0.1 * math.log(factor) + 1
    elif scaling == "bands":
        s = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0, 1)
        f = (1 - s) * f / factor + s * f
    a = np.arange(positions)[:, None] * f
    return np.stack([np.cos(a) * m, np.sin(a) * m], -1)


def attend(q, k, v, sees, scale):
    """One sequence in 64 bits: q [n, heads, d], k / v [length, kv_heads, d], sees [n, length].
    (out, lse, sum of p |v|, largest sum of |q| |k| scale seen by the row)."""
    n, heads, d = q.shape
    g = heads // k.shape[1]
    out, lse = np.zeros((n, heads, d)), np.full((n, heads), -np.inf)
    mag, dot = np.zeros((n, heads, d)), np.zeros((n, heads))
    for h in range(heads):
        for i in range(n):
            at = np.flatnonzero(sees[i])
            if len(at) == 0:
                continue
            kk, vv = k[at, h // g], v[at, h // g]
            s = kk @ q[i, h] * scale
            m = s.max()
            e = np.exp(s - m)
            out[i, h], lse[i, h] = e @ vv / e.sum(), m + np.log(e.sum())
            mag[i, h] = e @ np.abs(vv) / e.sum()
            dot[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
    return out, lse, mag, dot


def verify(logits, tokens, parents, temperature, uniform, noise, probs=None):
    """One sequence's tree in 64 bits: (path, next token)."""
    n, vocab = logits.shape

    def target(row):
        x = logits[row].astype(np.float64)
        x = np.minimum(np.where(np.isnan(x), -np.inf, x), float(np.finfo(F32).max))
        p = np.zeros(vocab)
        if x.max() == -np.inf:
            return p
        if not temperature > 0:
            p[x.argmax()] = 1
            return p
        with np.errstate(over="ignore"):
            e = np.exp((x - x.max()) / temperature)
        return e / e.sum()

    cur, path, left, spent = 0, [0], target(0), False
    for i in range(1, n):
        if (parents[i] if parents is not None else i - 1) != cur or spent:
            continue
        t = int(tokens[i])
        inside = 0 <= t < vocab
        greedy = not temperature > 0
        q = np.zeros(vocab) if probs is None or greedy else probs[cur].astype(np.float64)
        if (probs is None or greedy) and inside:
            rest = left.copy()
            rest[t], q[t] = 0, 1
        else:
            rest = np.maximum(left - q, 0)
        u = 0.0 if greedy else float(uniform[i])
        if inside and u * q[t] < left[t]:
            cur = i
            path.append(i)
            left = target(i)
        elif rest.sum() <= 0:
            left, spent = target(cur), True
        else:
            left = rest / rest.sum()
    with np.errstate(divide="ignore", invalid="ignore"):
        score = left if not temperature > 0 else np.where(left > 0, left / noise, 0)
    return path, int(score.argmax()) if score.max() > 0 else -1
