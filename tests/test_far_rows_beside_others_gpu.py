"""Attention by runs over both caches: rows whose scores are far from 0 beside rows of the same warp whose scores are not."""
import numpy as np
import pytest
import torch

import plain_kv4
import test_kv4_gpu as kv4
import test_kv8_gpu as kv8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mine", [700.0, 9_000.0, 40_000.0])
@pytest.mark.parametrize("heads,dim", [(4, 64), (8, 128), (12, 64), (24, 128), (2, 256)])
@pytest.mark.parametrize("cache", ["4 bits", "8 bits"])
def test_equal_keys_count_the_same_whatever_stands_beside_them(gpu, cache, heads, dim, mine):
    """The first head's keys are all the same in the first half of its dims, so its output is the mean of the values; the other heads' scores go far from 0 half-way."""
    rng = np.random.default_rng(dim)
    ctx, page = 331, 16
    n = ctx + 1
    four = cache == "4 bits"
    s = (kv4 if four else kv8).Setup(gpu, [(ctx, 1)], 1, dim, page, seed=dim)
    p, half, top = s.plain, dim // 2, 7 if four else 127
    key = np.zeros((n, dim), int)
    key[:, :half] = rng.integers(-top, top + 1, half)
    key[:, 0] = top
    key[n // 2:, half:] = top
    for slot in range(n):
        p.k[s.table[0, slot // page], 0, slot % page] = plain_kv4.pack(key[slot]) if four else key[slot]
    p.k_scale[:], p.v_scale[:] = 1.0, 0.0625
    if four:
        p.k_block[:], p.v_block[:] = 0x38, 0x38                # 1
    names = ("k", "v", "k_block", "v_block", "k_scale", "v_scale") if four else ("k", "v", "k_scale", "v_scale")
    for t, name in zip(s.pools, names):
        t.copy_(kv4.cuda(getattr(p, name)))
    q = np.zeros((1, heads, dim), np.float32)
    q[0, 0, :half] = np.sign(key[0, :half]) * rng.uniform(0.5, 1.0, half)
    q[0, 0] *= mine / float(key[0] @ q[0, 0].astype(np.float64))
    q[0, 1:, half:] = 1e7
    out = torch.empty(1, heads, dim, device="cuda")
    s.cache.attention(s.batch, torch.from_numpy(q).cuda(), out, scale=1.0)
    got = kv4.host(out)[0, 0].astype(np.float64)
    v = p.values("v", s.table[0], n)[:, 0]
    want, amp = v.mean(0), np.abs(v).mean(0)
    # Equal scores have equal weights, bit for bit: 22 bits of them are multiplied, sums are in f32 (2^-20), then a quotient, a product and the output's rounding.
    assert (np.abs(got - want) <= amp * 2.0 ** -19).all(), (np.abs(got - want) / amp).max() * 2 ** 19
    last = kv4.host(out)[0, 1:].astype(np.float64)
    want, amp = v[n // 2:].mean(0), np.abs(v[n // 2:]).mean(0)
    assert (np.abs(last - want) <= amp * 2.0 ** -19).all()
