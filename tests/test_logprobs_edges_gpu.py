"""Log probabilities of rows whose logits span more than f32's range, against the same in 64 bits."""
import math

import numpy as np
import pytest
import torch

import plain_kv8 as plain
from test_logprobs_gpu import DT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [40, 9000, 40000])
def test_spreads_beyond_the_types_range(gpu, dtype, vocab):
    """The type's lowest value and numbers near its largest in one row, in any order: the difference is an infinity, the entropy is not."""
    low, high = torch.finfo(DT[dtype]).min, 1e38
    g = torch.Generator().manual_seed(81)
    x = torch.randn(12, vocab, generator=g)
    x[0] = low
    x[0, vocab - 1] = high                                # the last of all
    x[1] = low
    x[1, 0] = high                                        # the first
    x[2] = low
    x[2, vocab // 2] = x[2, vocab // 2 + 1] = high        # two of them
    x[3, : vocab // 2] = low
    x[3, vocab // 2:] = high
    x[4, ::2] = low
    x[4, 1::2] = high
    x[5] = low
    x[6] = -1e38
    x[6, vocab // 3] = 3e38
    x[7, : vocab - 1] = low                               # one ordinary logit among them
    x[8] = torch.linspace(-3e38, 3e38, vocab, dtype=torch.float64)  # in f32 its step would be infinite
    x[9] = low
    x[9, vocab - 1] = math.inf                            # not finite: NaN
    x[10, : vocab // 4] = -math.inf
    x[10, vocab // 4: vocab // 2] = low
    x[10, vocab // 2:] = high
    x = x.to(DT[dtype]).cuda()
    tokens = torch.randint(vocab, (12,), generator=g).cuda()
    lp, ent, tl, ti = (a.cpu().numpy() for a in gpu.token_logprobs_dev(x, tokens, top=5))
    want = plain.logprobs(x.double().cpu().numpy(), tokens.cpu().numpy(), 5)
    assert np.isnan(ent).tolist() == [r == 9 for r in range(12)]
    assert np.array_equal(ti, want[3])
    # the bounds of the tests of ordinary rows; what lies below f32's range is minus infinity there
    off = 2.0 ** -20 + (16 + math.log(vocab)) * 2.0 ** -23
    for got, w, o in ((lp, want[0], off), (tl, want[2], off), (ent, want[1], off * (16 + math.log(vocab)))):
        with np.errstate(over="ignore"):
            w32 = w.astype(np.float32)
        assert np.array_equal(np.isnan(got), np.isnan(w32)) and np.array_equal(got == -np.inf, w32 == -np.inf)
        fine = np.isfinite(w32)
        assert (np.abs(got[fine] - w[fine]) <= o + np.abs(w[fine]) * 2.0 ** -23).all()
