"""The 8-bit key/value cache and log probabilities from their definitions, in 64 bits (numpy), a sequence and a page at a time."""
import math

import numpy as np

EPS = {"float32": 2.0 ** -23, "float16": 2.0 ** -10, "bfloat16": 2.0 ** -7}
TINY = {"float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0}  # half of f16's smallest step; the others' is below all test data


def rotation(turns, pos):
    """(cos, sin) of position times entry, the products taken as whole numbers modulo 2^64."""
    frac = np.array([(int(pos) * int(t)) % 2 ** 64 for t in turns], dtype=object)
    signed = np.array([f - 2 ** 64 if f >= 2 ** 63 else f for f in frac], dtype=object)
    angle = np.array([float(f) * 2.0 ** -64 for f in signed]) * (2.0 * math.pi)
    return np.cos(angle), np.sin(angle)


def rotate(x, turns, pos):
    """Rows [n, heads, dim] at positions `pos`."""
    y = np.array(x, np.float64)
    half = len(turns)
    for j, p in enumerate(pos):
        c, s = rotation(turns, p)
        a, b = y[j, :, :half].copy(), y[j, :, half:2 * half].copy()
        y[j, :, :half], y[j, :, half:2 * half] = a * c - b * s, a * s + b * c
    return y


class PlainCache:
    """Pools as numpy arrays: k, v int8 [pages, kv, page, dim], scales f32 [pages, kv]."""

    def __init__(self, k, v, k_scale, v_scale):
        self.k, self.v, self.k_scale, self.v_scale = k.copy(), v.copy(), k_scale.copy(), v_scale.copy()
        self.page = k.shape[2]

    def append(self, table, ctx, row_start, k, v, turns):
        for i in range(len(ctx)):
            r0, r1 = row_start[i], row_start[i + 1]
            pos = ctx[i] + np.arange(r1 - r0)
            self._rows(self.k, self.k_scale, table[i], pos, rotate(k[r0:r1], turns, pos))
            self._rows(self.v, self.v_scale, table[i], pos, np.array(v[r0:r1], np.float64))

    def _rows(self, pool, scale, table, pos, x):
        for number in dict.fromkeys(p // self.page for p in pos):
            here = np.nonzero(pos // self.page == number)[0]
            at, first = table[number], pos[here[0]] % self.page
            y = x[here]                                                    # [rows, kv, dim]
            mags = np.where(np.isfinite(y), np.abs(y), 0.0).max(axis=(0, 2))
            before = scale[at].copy() if first else np.zeros(pool.shape[1], np.float32)
            now = np.maximum(before, (mags / 127.0).astype(np.float32))
            for h in range(pool.shape[1]):
                if first and now[h] != before[h]:
                    old = pool[at, h, :first].astype(np.float64)
                    pool[at, h, :first] = np.rint(old * float(before[h]) / float(now[h])).astype(np.int8)
                if now[h] > 0:
                    with np.errstate(invalid="ignore"):
                        q = np.clip(np.rint(y[:, h] / float(now[h])), -127, 127)
                    q = np.where(np.isnan(y[:, h]), 0, q)
                else:
                    q = np.zeros_like(y[:, h])
                pool[at, h, first:first + len(here)] = q.astype(np.int8)
            scale[at] = now

    def values(self, which, table, n):
        """Positions 0 .. n - 1 of a sequence, [n, kv, dim]."""
        pool, scale = (self.k, self.k_scale) if which == "k" else (self.v, self.v_scale)
        pos = np.arange(n)
        at = np.asarray(table)[pos // self.page]
        return pool[at, :, pos % self.page].astype(np.float64) * scale[at].astype(np.float64)[:, :, None]

    def attention(self, table, ctx, row_start, q, scale=None, window=0):
        """(out, sums of weight times |value|, largest sum of |q k| * scale per row and head, keys per row)"""
        q = np.array(q, np.float64)
        rows, heads, dim = q.shape
        scale = scale or 1.0 / math.sqrt(dim)
        out, mass, big, keys = np.zeros_like(q), np.zeros_like(q), np.zeros((rows, heads)), np.zeros(rows)
        group = heads // self.k.shape[1]
        for i in range(len(ctx)):
            r0, n = row_start[i], row_start[i + 1] - row_start[i]
            if n == 0:
                continue
            k, v = self.values("k", table[i], ctx[i] + n), self.values("v", table[i], ctx[i] + n)
            for j in range(n):
                lo, hi = max(0, ctx[i] + j + 1 - window) if window else 0, ctx[i] + j + 1
                keys[r0 + j] = hi - lo
                for h in range(heads):
                    s = k[lo:hi, h // group] @ q[r0 + j, h] * scale
                    big[r0 + j, h] = (np.abs(k[lo:hi, h // group]) @ np.abs(q[r0 + j, h])).max() * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[r0 + j, h] = p @ v[lo:hi, h // group]
                    mass[r0 + j, h] = p @ np.abs(v[lo:hi, h // group])
        return out, mass, big, keys


def attention_bound(out, mass, big, keys, dim, dtype, split):
    """How far an output may be off.  A weight is off by a factor e^(+-d) for a score off by d, so an output by at most 2 d of its mass (the sum of
    weight times |value|), the denominator counted.  d: what the query loses beyond 22 bits, the matrix unit's additions (dim / 16
    of them, cut off at 2^-23 of the largest term), four roundings to f32, all of at most `big`; 2^ of f32: 2^-21.  A weight is held in 22
    bits (split), or rounded to f16: half a step, 2^-11, and 2^-25 below its normal range where the largest is 2^8.  Sums in f32 of steps and
    warps: 2^-20.  Then the output's own rounding, by way of f32."""
    d = big * (2.0 ** -22 + (dim / 16 + 4) * 2.0 ** -23) + 2.0 ** -21
    weight = 2.0 ** -22 if split else 2.0 ** -11
    eps = 2 * (d[..., None] + weight) + 2.0 ** -20
    low = 0.0 if split else 2.0 ** -33 * keys[:, None, None] * np.abs(mass).max(initial=1.0) * 8
    return mass * eps + low + np.abs(out) * (EPS[dtype] / 2 + 2.0 ** -23) + TINY[dtype]


def logprobs(x, tokens, top):
    """(logprob, entropy, top_logprob, top_id) of rows of logits."""
    x = np.array(x, np.float64)
    rows, vocab = x.shape
    lp, ent = np.full(rows, np.nan), np.full(rows, np.nan)
    tl, ti = np.full((rows, top), np.nan), np.full((rows, top), -1, np.int64)
    for r in range(rows):
        if np.isnan(x[r]).any() or (x[r] == np.inf).any():
            continue
        order = np.lexsort((np.arange(vocab), -x[r]))[:top]
        ti[r] = order
        m = x[r].max()
        if m == -np.inf:
            y = np.full(vocab, -np.inf)
            ent[r] = 0.0
        else:
            y = x[r] - m - math.log(np.exp(x[r] - m).sum())
            p = np.exp(y)
            ent[r] = -(p[p > 0] * y[p > 0]).sum()
        tl[r] = y[order]
        if 0 <= tokens[r] < vocab:
            lp[r] = y[tokens[r]]
    return lp, ent, tl, ti
