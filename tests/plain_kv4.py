"""The 4-bit key/value cache, rotations, the weights of keys and eviction from their definitions, in 64 bits (numpy), a sequence and a head at a time."""
import math

import numpy as np

EPS = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}      # half a step
TINY = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}  # half a step of the smallest numbers (f32: a whole one)

# all e4m3 numbers without a sign, 0x7f among them as the 480 that its bits say
E4M3 = np.array([(c % 8) * 2.0 ** -9 if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7) for c in range(128)])


def angles(turns, pos):
    """position times entry, the products taken as whole numbers modulo 2^64, in radians: [positions, pairs]"""
    out = np.empty((len(pos), len(turns)))
    for i, p in enumerate(pos):
        for j, t in enumerate(turns):
            f = int(p) * int(t) % 2 ** 64
            out[i, j] = (f - 2 ** 64 if f >= 2 ** 63 else f) * 2.0 ** -64
    return out * (2.0 * math.pi)


def rotate(x, turns, pos, layout="half", magnitude=1.0, inverse=False):
    """Rows [n, heads, dim] at positions `pos`."""
    y = np.array(x, np.float64)
    n = len(turns)
    a = angles(turns, pos)
    c, s = np.cos(a)[:, None] * magnitude, np.sin(a)[:, None] * (-magnitude if inverse else magnitude)
    first, second = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    u, w = y[..., first].copy(), y[..., second].copy()
    y[..., first], y[..., second] = u * c - w * s, u * s + w * c
    return y


def quantise(x, g):
    """Integers and e4m3 codes of x [..., dim] under a head's scale g."""
    x = np.asarray(x, np.float64)
    blocks = x.reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    top = np.where(np.isfinite(blocks), np.abs(blocks), 0.0).max(-1)
    want = top / (7.0 * float(g))
    grid = E4M3[:127]
    up = np.clip(np.searchsorted(grid, want), 1, 126)
    low, high = grid[up - 1], grid[up]
    code = np.where((want - low < high - want) | ((want - low == high - want) & ((up - 1) % 2 == 0)), up - 1, up)
    step = (grid[code] * float(g))[..., None]
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.clip(np.rint(blocks / step), -7, 7)
    ints = np.where(np.isnan(blocks) | (step == 0), 0, np.nan_to_num(q)).astype(np.int8)
    return ints.reshape(x.shape), code.astype(np.uint8)


def pack(ints):
    u = (ints + 8).astype(np.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def unpack(packed):
    return np.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], -1).astype(np.float64) - 8.0


class PlainCache:
    """Pools as numpy arrays: k, v uint8 [pages, kv, page, dim / 2], blocks uint8 [pages, kv, page, dim / 16], scales f32 [kv]."""

    def __init__(self, k, v, k_block, v_block, k_scale, v_scale):
        self.k, self.v, self.k_block, self.v_block, self.k_scale, self.v_scale = (a.copy() for a in (k, v, k_block, v_block, k_scale, v_scale))
        self.page = k.shape[2]

    def append(self, table, ctx, row_start, k, v, turns, positions=None, layout="half", magnitude=1.0):
        for i in range(len(ctx)):
            r0, r1 = row_start[i], row_start[i + 1]
            slot, j = ctx[i] + np.arange(r1 - r0), np.arange(r1 - r0)
            pos = slot if positions is None else positions[i] + j
            new = {"k": rotate(k[r0:r1], turns, pos, layout, magnitude) if len(turns) else np.asarray(k[r0:r1], np.float64), "v": np.asarray(v[r0:r1], np.float64)}
            at = np.asarray(table[i])[slot // self.page]
            for name, x in new.items():
                for h in range(self.k.shape[1]):
                    ints, code = quantise(x[:, h], getattr(self, name + "_scale")[h])
                    getattr(self, name)[at, h, slot % self.page] = pack(ints)
                    getattr(self, name + "_block")[at, h, slot % self.page] = code

    def values(self, which, table, n):
        """Slots 0 .. n - 1 of a sequence, [n, kv, dim]."""
        slot = np.arange(n)
        at = np.asarray(table)[slot // self.page]
        ints = unpack(getattr(self, which)[at, :, slot % self.page])
        block = E4M3[getattr(self, which + "_block")[at, :, slot % self.page] & 127].repeat(16, -1)
        return ints * block * getattr(self, which + "_scale").astype(np.float64)[None, :, None]

    def attention(self, table, ctx, row_start, q, scale=None, window=0):
        """(out, lse, sums of weight times |value|, largest sum of |q k| * scale per row and head, keys per row, weights [(seq, row, head, first slot, p)])"""
        q = np.array(q, np.float64)
        rows, heads, dim = q.shape
        scale = scale or 1.0 / math.sqrt(dim)
        out, mass, big, keys, lse, weights = np.zeros_like(q), np.zeros_like(q), np.zeros((rows, heads)), np.zeros(rows), np.full((rows, heads), np.nan), []
        group = heads // self.k.shape[1]
        for i in range(len(ctx)):
            r0, n = row_start[i], row_start[i + 1] - row_start[i]
            if n <= 0:
                continue
            k, v = self.values("k", table[i], ctx[i] + n), self.values("v", table[i], ctx[i] + n)
            for j in range(n):
                lo, hi = max(0, ctx[i] + j + 1 - window) if window else 0, ctx[i] + j + 1
                keys[r0 + j] = hi - lo
                for h in range(heads):
                    s = k[lo:hi, h // group] @ q[r0 + j, h] * scale
                    big[r0 + j, h] = (np.abs(k[lo:hi, h // group]) @ np.abs(q[r0 + j, h])).max() * scale
                    p = np.exp(s - s.max())
                    lse[r0 + j, h] = s.max() + math.log(p.sum())
                    p /= p.sum()
                    out[r0 + j, h] = p @ v[lo:hi, h // group]
                    mass[r0 + j, h] = p @ np.abs(v[lo:hi, h // group])
                    weights.append((i, r0 + j, h, lo, p))
        return out, lse, mass, big, keys, weights


def score_bound(big, dim):
    """How far a score (times its scale) may be off: what the query loses beyond 22 bits, the matrix unit's additions (dim / 16 of them, cut off at 2^-23 of the largest term), six roundings
    to f32, all of at most `big`; and 2^ of f32: 2^-21."""
    return big * (2.0 ** -22 + (dim / 16 + 6) * 2.0 ** -23) + 2.0 ** -21


def attention_bound(out, mass, big, keys, dim, dtype, split):
    """How far an output may be off.  A weight is off by a factor e^(+-d) for a score off by d, so an output by at most 2 d of its mass (the sum of
    weight times |value|), the denominator counted.  A weight is held in 22 bits (split), or rounded to f16: half a step, 2^-11.  In both forms nothing below f16's smallest step, 2^-24, is
    held, half of which a weight may lose, where the row's largest is 2^6 or more (2^10 where few rows make a sequence): 2^-31 of it, times a value, for which the largest mass stands (a split form
    without this part asks for weights of 1e-39 beside one of 1).  Sums in f32 of steps and warps: 2^-20.  Then the output's own rounding, by way of f32."""
    d = score_bound(big, dim)
    weight = 2.0 ** -22 if split else 2.0 ** -11
    eps = 2 * (d[..., None] + weight) + 2.0 ** -20
    low = 2.0 ** -31 * keys[:, None, None] * np.abs(mass).max(initial=1.0)
    return mass * eps + low + np.abs(out) * (EPS[dtype] + 2.0 ** -23) + TINY[dtype]


def evict(mass, length, keep, limit, recent, first):
    """Slots that stay of sums [length] (all, where there are not more than limit), in ascending order."""
    if length <= limit:
        return np.arange(length)
    w = np.where(np.isnan(mass[:length]), -np.inf, mass[:length].astype(np.float64)) + 0.0
    inner = np.arange(first, length - recent)
    order = inner[np.lexsort((inner, -w[inner]))]
    # NaN behind everything, minus infinity too: the lower slot first among them only if both are NaN or both are not
    order = np.array(sorted(order, key=lambda x: (np.isnan(mass[x]), -w[x], x)), int)
    return np.sort(np.concatenate((np.arange(first), order[:keep - first - recent], np.arange(length - recent, length))).astype(int))
