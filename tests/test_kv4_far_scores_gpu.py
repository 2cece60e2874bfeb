"""Attention over the 4-bit cache with scores so far from 0 that neighbouring f32 numbers are 4, 8 or 16 powers of two apart: two keys whose scores are neighbours, the lower one first."""
import numpy as np
import pytest
import torch

import plain_kv4 as plain
from test_kv4_gpu import DT, Setup, cuda, host

pytestmark = pytest.mark.gpu

LN2 = float(np.float32(np.log(2.0)))   # times log2 e it is 1 in f32: scores are then whole numbers of powers of two


def neighbours(gpu, dtype, exponent, sign, kv, heads, dim, rows, first, second):
    """A sequence whose keys in the slots `first` and `second` have scores of +-2^exponent or a little more, the second's one f32 step above the first's; all other keys are far below.
    Head h of the kv heads begins h steps higher, so that odd and even multiples of the step stand first.  Returns what attention gave and what the two keys' values give."""
    step = 2.0 ** (exponent - 23)
    ctx = second + 17
    s = Setup(gpu, [(ctx, rows)], kv, dim, 16, seed=exponent + dim)
    # integers of the first dims times 256, of dims 16 and up times 1; four numbers of 2^(exponent - 2) make the score, dim 16 the steps
    ints = np.zeros((ctx + rows, kv, dim), int)
    ints[:, :, :4] = -7
    for h in range(kv):
        for slot, more in ((first, h + 1 if sign > 0 else -h - 2), (second, h + 2 if sign > 0 else -h - 1)):
            ints[slot, h, :4], ints[slot, h, 16] = 4 * sign, more
    value = np.zeros((ctx + rows, kv, dim), int)
    value[first, :, 0::2], value[second, :, 1::2] = 7, 5
    p = s.plain
    p.k_scale[:] = p.v_scale[:] = 1.0
    p.k_block[:], p.v_block[:] = 0x38, 0x38                     # 1
    p.k_block[..., 0] = 0x78                                    # 256
    for slot in range(ctx + rows):
        p.k[s.table[0, slot // 16], :, slot % 16] = plain.pack(ints[slot])
        p.v[s.table[0, slot // 16], :, slot % 16] = plain.pack(value[slot])
    for t, a in zip(s.pools, (p.k, p.v, p.k_block, p.v_block, p.k_scale, p.v_scale)):
        t.copy_(cuda(a))
    q = torch.zeros(rows, heads, dim)
    q[:, :, :4] = 2.0 ** (exponent - 12)
    q[:, :, 16] = step
    q = q.to(DT[dtype])
    q64 = q.double().numpy()
    k = p.values("k", s.table[0], ctx + rows)
    score = np.einsum("rhd,khd->rhk", q64, k.repeat(heads // kv, 1))
    two = score[:, :, [first, second]]
    assert (two == two.astype(np.float32)).all() and (two[..., 1] - two[..., 0] == step).all() and (np.delete(score, [first, second], -1) < two[..., :1] - 1e6).all()
    assert (np.abs(two) >= 2.0 ** exponent).all() and (np.abs(two) < 2.0 ** (exponent + 1)).all()
    out, lse = torch.empty_like(q, device="cuda"), torch.empty(rows, heads, device="cuda")
    s.cache.attention(s.batch, q.cuda(), out, lse=lse, scale=LN2)
    want = np.zeros((rows, heads, dim))
    want[..., 0::2], want[..., 1::2] = 7.0 / (1.0 + 2.0 ** step), 5.0 / (1.0 + 2.0 ** -step)
    return host(out).astype(np.float64), want, host(lse).astype(np.float64), two[..., 1] * LN2


def check(dtype, out, want, lse, wlse):
    # Scores, their differences and both weights, powers of two, are exact.  What is left: two exponentials of the chip (2^-22 each), a sum, a quotient and a product in f32, the output's own rounding.
    assert (np.abs(out - want) <= want * (plain.EPS[dtype] + 2.0 ** -20)).all()
    # the logarithm's sum and product in f32, two roundings
    assert (np.abs(lse - wlse) <= np.abs(wlse) * 2.0 ** -23).all()


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("exponent", [25, 26, 27])
@pytest.mark.parametrize("sign", [1, -1], ids=["above", "below"])
@pytest.mark.parametrize("kv,heads,dim,rows", [(2, 8, 64, 1), (2, 4, 128, 1), (2, 32, 128, 1), (2, 8, 64, 6), (2, 8, 128, 5), (2, 4, 256, 1), (2, 12, 256, 2), (2, 2, 80, 3)], ids=str)
def test_neighbouring_scores_far_from_zero_in_runs(gpu, dtype, exponent, sign, kv, heads, dim, rows):
    check(dtype, *neighbours(gpu, dtype, exponent, sign, kv, heads, dim, rows, 3, 20))


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("exponent", [25, 26, 27])
@pytest.mark.parametrize("sign", [1, -1], ids=["above", "below"])
@pytest.mark.parametrize("kv,heads,dim,rows", [(2, 4, 64, 70), (2, 8, 128, 40), (2, 2, 112, 300)], ids=str)
@pytest.mark.parametrize("second", [20, 150])
def test_neighbouring_scores_far_from_zero_in_tiles(gpu, dtype, exponent, sign, kv, heads, dim, rows, second):
    check(dtype, *neighbours(gpu, dtype, exponent, sign, kv, heads, dim, rows, 3, second))
