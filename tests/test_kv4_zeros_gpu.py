"""Appends of zeros to the 4-bit cache: rows that fill up a batch, heads that are switched off, blocks of zeros in front of and behind others, of either sign, turned or not."""
import numpy as np
import pytest
import torch

from test_kv4_gpu import DT, Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("layout,rot", [("half", 0), ("half", 96), ("interleaved", 64), ("half", 20)])
def test_zeros_among_other_numbers(gpu, dtype, layout, rot):
    s = Setup(gpu, [(3, 70), (40, 9)], 3, 96, 16, seed=rot)
    (k, _), (v, _) = s.normal(3, dtype), s.normal(3, dtype)
    for t in (k, v):
        t[::3] = 0.0
        t[1::5, 1] = 0.0
        t[2::4, :, 16:48] = -0.0
        t[5, 0, 17:32] = 0.0                                    # but one
        t[6, 2, 0:16], t[6, 2, 3] = 0.0, float("nan")
        t[7, 2, 0:16], t[7, 2, 3] = 0.0, float("inf")
    turns, on_gpu = s.turns(rot)
    s.cache.append(s.batch, k, v, turns=on_gpu if rot else None, layout=layout)
    k64, v64 = (t.double().cpu().numpy() for t in (k, v))
    with np.errstate(invalid="ignore"):
        s.plain.append(s.table, s.ctx, s.start, k64, v64, turns, layout=layout)
    s.check_pools()


def test_rows_of_zeros_take_no_longer_than_others(gpu):
    """By the clock, with a wide margin: they took seven times as long when every block of zeros was looked at in 64 bits."""
    s = Setup(gpu, [(0, 4096)], 8, 128, 64, seed=1)
    k, v = s.normal(8, "bfloat16")[0], s.normal(8, "bfloat16")[0]
    _, on_gpu = s.turns(128)
    times = []
    for some in (k, torch.where(torch.arange(4096, device="cuda")[:, None, None] % 8 == 0, 0.0, k).to(k.dtype)):
        took = []
        for _ in range(15):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            begin.record()
            for _ in range(10):
                s.cache.append(s.batch, some, v, turns=on_gpu)
            end.record()
            torch.cuda.synchronize()
            took.append(begin.elapsed_time(end))
        times.append(np.median(took))
    assert times[1] < 2 * times[0], times
