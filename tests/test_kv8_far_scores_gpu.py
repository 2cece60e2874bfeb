"""Attention over the 8-bit cache with scores so far from 0 that neighbouring f32 numbers are 4, 8 or 16 powers of two apart: two keys whose scores are neighbours, the lower one first."""
import numpy as np
import pytest
import torch

import plain_kv8 as plain
from test_kv8_gpu import DT, Setup, cuda, host

pytestmark = pytest.mark.gpu

LN2 = float(np.float32(np.log(2.0)))   # times log2 e it is 1 in f32


def neighbours(gpu, dtype, exponent, sign, kv, heads, dim, rows, first, second, louder):
    """A sequence whose keys in the slots `first` and `second` have scores between +-2^exponent and twice that, the second's one f32 step above the first's; all other keys are far below.  Head h of the kv
    heads begins h steps higher, so that odd and even multiples of the step stand first; the second key's page has values `louder` times as large.  Returns what attention gave and what it should."""
    step = 2.0 ** (exponent - 23)
    ctx = second + 17
    s = Setup(gpu, [(ctx, rows)], kv, dim, 16, seed=exponent + dim)
    k = np.zeros((ctx + rows, kv, dim), int)
    k[:, :, :3] = -127
    for h in range(kv):
        for slot, more in ((first, h + 1 if sign > 0 else -h - 2), (second, h + 2 if sign > 0 else -h - 1)):
            k[slot, h, :3], k[slot, h, 16] = 127 if sign > 0 else -87, more
    value = np.zeros((ctx + rows, kv, dim), int)
    value[first, :, 0::2], value[second, :, 1::2] = 100, 90
    p = s.plain
    p.k_scale[:], p.v_scale[:] = step, 1.0
    p.v_scale[s.table[0, second // 16]] = louder
    for slot in range(ctx + rows):
        p.k[s.table[0, slot // 16], :, slot % 16] = k[slot]
        p.v[s.table[0, slot // 16], :, slot % 16] = value[slot]
    for t, a in zip(s.pools, (p.k, p.v, p.k_scale, p.v_scale)):
        t.copy_(cuda(a))
    q = torch.zeros(rows, heads, dim)
    q[:, :, :3], q[:, :, 16] = 127.0 * 256.0, 1.0               # whole numbers of a row's largest / (127 x 256)
    q = q.to(DT[dtype])
    score = np.einsum("rhd,khd->rhk", q.double().numpy(), p.values("k", s.table[0], ctx + rows).repeat(heads // kv, 1))
    two = score[:, :, [first, second]]
    assert (two == two.astype(np.float32)).all() and (two[..., 1] - two[..., 0] == step).all() and (np.delete(score, [first, second], -1) < two[..., :1] - 1e6).all()
    assert (np.abs(two) >= 2.0 ** exponent).all() and (np.abs(two) < 2.0 ** (exponent + 1)).all()
    out = torch.empty_like(q, device="cuda")
    s.cache.attention(s.batch, q.cuda(), out, scale=LN2)
    want = np.zeros((rows, heads, dim))
    want[..., 0::2], want[..., 1::2] = 100.0 / (1.0 + 2.0 ** step), 90.0 * louder / (1.0 + 2.0 ** -step)
    return host(out).astype(np.float64), want


def check(dtype, out, want):
    # Scores, their differences and both weights, powers of two, are exact (EPS is a whole step here).  What is left: two exponentials of the chip (2^-22 each), the scales' quotient, a sum, a quotient and
    # a product in f32, the output's own rounding.
    assert (np.abs(out - want) <= want * (plain.EPS[dtype] / 2 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("exponent", [24, 25, 26, 27])
@pytest.mark.parametrize("sign,louder", [(1, 1.0), (-1, 1.0), (1, 16.0), (-1, 0.125)], ids=["above", "below", "above loud", "below quiet"])
@pytest.mark.parametrize("kv,heads,dim,rows", [(2, 8, 64, 1), (2, 4, 128, 1), (2, 32, 128, 1), (2, 8, 64, 6), (2, 8, 128, 5), (2, 4, 256, 1), (2, 12, 256, 2), (2, 2, 80, 3)], ids=str)
def test_neighbouring_scores_far_from_zero_in_runs(gpu, dtype, exponent, sign, louder, kv, heads, dim, rows):
    check(dtype, *neighbours(gpu, dtype, exponent, sign, kv, heads, dim, rows, 3, 20, louder))


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("exponent", [24, 25, 26, 27])
@pytest.mark.parametrize("sign,louder", [(1, 1.0), (-1, 1.0), (1, 16.0), (-1, 0.125)], ids=["above", "below", "above loud", "below quiet"])
@pytest.mark.parametrize("kv,heads,dim,rows", [(2, 4, 64, 70), (2, 8, 128, 40), (2, 2, 112, 300), (8, 16, 128, 150)], ids=str)
@pytest.mark.parametrize("second", [20, 150])
def test_neighbouring_scores_far_from_zero_in_tiles(gpu, dtype, exponent, sign, louder, kv, heads, dim, rows, second):
    check(dtype, *neighbours(gpu, dtype, exponent, sign, kv, heads, dim, rows, 3, second, louder))


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("exponent", [10, 16, 22, 28, 30, 45])
@pytest.mark.parametrize("kv,heads,dim,seqs", [(2, 8, 64, [(600, 40), (130, 70)]), (2, 2, 128, [(3000, 150)]), (8, 32, 48, [(200 + 7 * i, 32) for i in range(20)]), (2, 4, 64, [(600, 2)])], ids=["cut", "cut long", "whole", "few"])
def test_equal_scores_far_from_zero_of_pages_of_other_scales(gpu, dtype, exponent, kv, heads, dim, seqs):
    """Keys that are all the same, or the opposite: a row's output is the mean of the values of those that it likes, on pages whose scales are far apart."""
    rng = np.random.default_rng(exponent)
    s = Setup(gpu, seqs, kv, dim, 16, seed=dim)
    p = s.plain
    key = rng.integers(-127, 128, (kv, dim))
    key[:, 0] = 127
    p.k_scale[:] = 2.0 ** -7
    p.v_scale[:] = np.exp2(rng.uniform(-8, 8, p.v_scale.shape)).astype(np.float32)
    signs = []
    for i, (c, n) in enumerate(seqs):
        sign = np.where(rng.random((c + n, kv)) < 0.3, 1, -1)
        sign[0] = 1
        for slot in range(c + n):
            p.k[s.table[i, slot // 16], :, slot % 16] = sign[slot][:, None] * key
        signs.append(sign)
    for t, a in zip(s.pools, (p.k, p.v, p.k_scale, p.v_scale)):
        t.copy_(cuda(a))
    # queries along the key or against it, each of its own size up to a factor of 4
    q = np.sign(key).repeat(heads // kv, 0)[None] * np.abs(rng.normal(0, 1, (s.rows, heads, dim))) * np.exp2(rng.uniform(0, 2, (s.rows, heads, 1)))
    q = torch.from_numpy((q * np.where(rng.random((s.rows, heads, 1)) < 0.8, 1, -1)).astype(np.float32)).to(DT[dtype])
    q64 = q.double().numpy()
    out = torch.empty_like(q, device="cuda")
    s.cache.attention(s.batch, q.cuda(), out, scale=2.0 ** (exponent - 8))
    got, clear, seen = host(out).astype(np.float64), 0, 0
    for i, (c, n) in enumerate(seqs):
        v = p.values("v", s.table[i], c + n)
        for j in range(0, n, 1 + n // 16):
            for h in range(heads):
                g, r = h // (heads // kv), int(s.start[i]) + j
                score = float(key[g] @ q64[r, h]) * 2.0 ** (exponent - 15)
                seen += 1
                mine = signs[i][:c + j + 1, g] * score > 0
                if not mine.any():
                    mine = ~mine
                elif 2 * abs(score) < 200.0:
                    continue                                    # the others would count as well
                clear += 1
                some = v[:c + j + 1, g][mine]
                want, amp = some.mean(0), np.abs(some).mean(0)
                # All weights are the same.  Each is off by its exponential, its scale's logarithm (2^-22 of up to 8) and its rounding to 11 bits (f32: 22), or by 2^-31 of the largest weight and scale;
                # sums in f32, then the output's own rounding.  Near 0 (scores of up to 2^16 powers of two) log2 of a page's scale, 6 and the reference m are added up in f32 before the score is: two
                # roundings of 2^-24 m each, which differ between pages, so a weight is off by ln 2 x 2^-23 m and an output, numerator and denominator, by twice that, 1.4 x 2^-23 m.
                m = abs(score) * 1.4427
                near = m * 2.0 ** -22 if m < 65600.0 else 0.0
                bound = amp * (2.0 ** -18 + (dtype != "float32") * 2.0 ** -10 + near) + np.abs(v[:c + j + 1, g]).max() * 2.0 ** -31 + np.abs(want) * plain.EPS[dtype] / 2 + plain.TINY[dtype]
                assert (np.abs(got[r, h] - want) <= bound).all(), (r, h, (np.abs(got[r, h] - want) / bound).max())
    assert clear > seen / 2


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("exponent", [17, 20, 30])
@pytest.mark.parametrize("kv,heads,seqs", [(2, 4, [(300, 300), (390, 150)]), (8, 32, [(380, 40)] * 20), (2, 4, [(420, 3), (390, 2)])], ids=["cut", "whole", "few"])
def test_scores_that_come_near_and_go_far_again(gpu, dtype, exponent, kv, heads, seqs):
    """Keys far below 0 in the first 256 slots, keys of 0 up to slot 400, keys far above 0 from there: a row's output is the mean of the last kind's values that it sees."""
    dim = 64
    rng = np.random.default_rng(exponent)
    s = Setup(gpu, seqs, kv, dim, 16, seed=dim)
    p = s.plain
    key = rng.integers(-127, 128, (kv, dim))
    key[:, 0] = 127
    p.k_scale[:] = 2.0 ** -7
    p.v_scale[:] = np.exp2(rng.uniform(-8, 8, p.v_scale.shape)).astype(np.float32)
    for i, (c, n) in enumerate(seqs):
        for slot in range(c + n):
            p.k[s.table[i, slot // 16], :, slot % 16] = key * (-1 if slot < 256 else 0 if slot < 400 else 1)
    for t, a in zip(s.pools, (p.k, p.v, p.k_scale, p.v_scale)):
        t.copy_(cuda(a))
    q = torch.from_numpy((np.sign(key).repeat(heads // kv, 0)[None] * np.abs(rng.normal(0, 1, (s.rows, heads, dim)))).astype(np.float32)).to(DT[dtype])
    out = torch.empty_like(q, device="cuda")
    s.cache.attention(s.batch, q.cuda(), out, scale=2.0 ** (exponent - 5))
    got = host(out).astype(np.float64)
    for i, (c, n) in enumerate(seqs):
        v = p.values("v", s.table[i], c + n)
        for j in range(0, n, 1 + n // 16):
            for h in range(heads):
                g, r, end = h // (heads // kv), int(s.start[i]) + j, c + j + 1
                some = v[400 if end > 400 else 256:end, g]
                want, amp = some.mean(0), np.abs(some).mean(0)
                # as above, the weights that count have scores of 0 or far ones
                bound = amp * (2.0 ** -18 + (dtype != "float32") * 2.0 ** -10) + np.abs(v[:end, g]).max() * 2.0 ** -31 + np.abs(want) * plain.EPS[dtype] / 2 + plain.TINY[dtype]
                assert (np.abs(got[r, h] - want) <= bound).all(), (r, h, (np.abs(got[r, h] - want) / bound).max())
