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
