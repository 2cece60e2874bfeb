"""Rotations in f32 of pairs that nearly cancel: what is left of two products is far smaller than they are."""
import numpy as np
import pytest
import torch

import plain_kv4 as plain
from test_rope_gpu import table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("magnitude", [1.0, 1.3])
@pytest.mark.parametrize("inverse", [False, True], ids=["forward", "back"])
@pytest.mark.parametrize("second", [False, True], ids=["first", "second"])
def test_pairs_that_cancel(gpu, layout, magnitude, inverse, second):
    rows, rot, tries = 40, 32, 4096
    rng = np.random.default_rng(7)
    turns, on_gpu = table(gpu, rot)
    pos = rng.integers(1, 2 ** 20, rows)
    a = plain.angles(turns, pos)
    c, s = np.cos(a), np.sin(a) * (-1.0 if inverse else 1.0)
    # of many f32 numbers u, and w = the f32 number next to what would make u c - w s (or u s + w c) 0, the pair that leaves least
    u = rng.normal(0, 1, (tries, rows, rot // 2)).astype(np.float32).astype(np.float64)
    w = (u * (-s / c if second else c / s)).astype(np.float32).astype(np.float64)
    left = np.abs(u * s + w * c if second else u * c - w * s) / np.hypot(u, w)
    best = left.argmin(0)
    u, w, left = (np.take_along_axis(t, best[None], 0)[0] for t in (u, w, left))
    assert np.median(left) < 2.0 ** -34
    x = np.zeros((rows, 1, rot), np.float32)
    one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    x[:, 0, one], x[:, 0, two] = u, w
    got = gpu.rope_dev(torch.from_numpy(x).cuda(), torch.from_numpy(pos).cuda(), on_gpu, layout=layout, magnitude=magnitude, inverse=inverse).double().cpu().numpy()
    want = plain.rotate(x, turns, pos, layout, magnitude, inverse)
    length = np.hypot(u, w) * magnitude
    # Sine and cosine as two f32 (the second 2^-48 of them off), the second parts' products and the sums of what was lost (2^-24 of 2^-24 of the products each, 7 x 2^-48 of the pair's length together),
    # the difference's and the last sum's rounding: 2^-23 of the result.
    bound = np.zeros_like(want)
    for part in (one, two):
        bound[:, 0, part] = np.abs(want[:, 0, part]) * 2.0 ** -22 + length * 2.0 ** -45
    assert (np.abs(got - want) <= bound).all()
