"""Log probabilities of given tokens, entropies and likeliest tokens against the same in 64 bits."""
import math

import numpy as np
import pytest
import torch

import plain_kv8 as plain

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def host(t):
    return t.cpu().numpy()


def check(gpu, x, tokens, top, **kw):
    """x: a tensor on the GPU.  Bounds: a term e^d is off by 2^-22 and by what d's product with log2 e loses, |d| 2^-23; S by as much of
    itself (|d| weighted by e^d is below 16 + log of the vocabulary), so log S by that, plus the f32 sums of sixteen, 2^-20; T / S by the
    spread of d as well.  The output's rounding is 2^-24 of it."""
    x64 = x.double().cpu().numpy()
    want = plain.logprobs(x64, host(tokens), top)
    lp, ent, tl, ti = gpu.token_logprobs_dev(x, tokens, top=top, **kw)
    off = 2.0 ** -20 + (16 + math.log(x.shape[1])) * 2.0 ** -23
    for got, w, o in ((lp, want[0], off), (tl, want[2], off), (ent, want[1], off * (16 + math.log(x.shape[1])))):
        got = host(got).astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(w))
        assert np.array_equal(got == -np.inf, w == -np.inf)
        fine = np.isfinite(w)
        assert (np.abs(got[fine] - w[fine]) <= o + np.abs(w[fine]) * 2.0 ** -23).all()
    assert np.array_equal(host(ti), want[3])
    return lp, ent, tl, ti


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,vocab,top", [(1, 32000, 5), (1, 1, 1), (3, 7, 7), (64, 1000, 20), (2, 128256, 32), (700, 33, 32), (5, 4097, 0), (40, 2049, 3), (1, 65537, 1), (300, 9001, 10)])
def test_against_64_bits(gpu, dtype, rows, vocab, top):
    g = torch.Generator().manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(DT[dtype]).cuda()
    tokens = torch.randint(vocab, (rows,), generator=g).cuda()
    check(gpu, x, tokens, top)


@pytest.mark.parametrize("dtype", list(DT))
def test_rows_with_gaps_and_odd_alignment(gpu, dtype):
    g = torch.Generator().manual_seed(1)
    wide = (torch.randn(30, 5003, generator=g) * 2).to(DT[dtype]).cuda()
    tokens = torch.randint(4000, (30,), generator=g).cuda()
    for a, b in ((0, 5000), (1, 4997), (3, 4003)):
        check(gpu, wide[:, a:b], tokens[:].clamp(max=b - a - 1), 6)
    check(gpu, wide[::3, 8:4808], tokens[::3].contiguous(), 2)


@pytest.mark.parametrize("dtype", list(DT))
def test_ties_go_to_the_lower_index(gpu, dtype):
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-3, 4, (12, 40000), generator=g).to(DT[dtype]).cuda()
    x[3] = 1.5
    x[4, ::2], x[4, 1::2] = 0.0, -0.0
    check(gpu, x, torch.zeros(12, dtype=torch.int64).cuda(), 32)
    up = torch.arange(20000, dtype=torch.float32)[None].expand(3, -1).to(DT[dtype]).cuda()  # ever larger, in bf16 and f16 with ties
    check(gpu, up[:, :60000].clone(), torch.zeros(3, dtype=torch.int64).cuda(), 17)


def test_masks_infinities_and_nan(gpu):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(12, 9000, generator=g) * 4
    x[0, :] = -math.inf                                   # nothing left
    x[1, 1:] = -math.inf                                  # one token
    x[2, 100:] = -math.inf
    x[3, 17] = math.nan
    x[4, 8999] = math.inf
    x[5, :] = torch.finfo(torch.float32).min              # a mask of the type's lowest value everywhere
    x[6, 5:] = torch.finfo(torch.float32).min
    x[7, :4500] = -math.inf
    x[8] *= 1e30
    x[9, 3] = 60.0                                        # nearly certain
    x[10, 7:9] = -math.inf
    tokens = torch.tensor([3, 0, 50, 3, 3, 8, 2, 6000, 3, 3, 7, -1])
    lp, ent, tl, ti = check(gpu, x.cuda(), tokens.cuda(), 5)
    assert host(lp)[0] == -math.inf and host(ent)[0] == 0 and host(ti)[0].tolist() == [0, 1, 2, 3, 4]
    assert math.isnan(lp[3]) and math.isnan(ent[4]) and (ti[3] == -1).all()
    assert math.isnan(lp[11]) and not math.isnan(ent[11])


def test_tokens_outside_the_vocabulary(gpu):
    x = torch.zeros(4, 50).cuda()
    lp, ent, tl, ti = gpu.token_logprobs_dev(x, torch.tensor([-1, 50, 2 ** 40, 49]).cuda())
    assert torch.isnan(lp[:3]).all() and abs(lp[3].item() + math.log(50)) < 1e-5
    assert top_shape(tl) == top_shape(ti) == (4, 0)


def top_shape(t):
    return tuple(t.shape)


def test_host_form(gpu):
    rng = np.random.default_rng(4)
    x = rng.normal(0, 2, (6, 777)).astype(np.float32)
    tokens = rng.integers(0, 777, 6)
    lp, ent, tl, ti = gpu.token_logprobs(x, tokens, 9)
    d = gpu.token_logprobs_dev(torch.from_numpy(x).cuda(), torch.from_numpy(tokens).cuda(), top=9)
    for a, b in zip((lp, ent, tl, ti), d):
        assert np.array_equal(a, host(b))
    assert [a.shape for a in gpu.token_logprobs(x[:0], tokens[:0], 2)] == [(0,), (0,), (0, 2), (0, 2)]


def test_streams_graphs_and_outputs_of_the_callers(gpu):
    x = torch.randn(3, 5000, generator=torch.Generator().manual_seed(5)).cuda()
    tokens = torch.tensor([1, 2, 3]).cuda()
    want = gpu.token_logprobs_dev(x, tokens, top=4)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = gpu.token_logprobs_dev(x, tokens, *[torch.empty_like(w) for w in want], stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    out = [torch.empty_like(w) for w in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.token_logprobs_dev(x, tokens, *out)
    y = torch.randn(3, 5000, generator=torch.Generator().manual_seed(6)).cuda()
    keep = x.clone()
    x.copy_(y)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, gpu.token_logprobs_dev(y, tokens, top=4)))
    x.copy_(keep)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_many_rows_and_far_offsets(gpu):
    """Rows whose offsets pass 2^31 elements."""
    x = torch.zeros(2 ** 31 // 40000 + 5, 40000, dtype=torch.float16, device="cuda")
    x[-1, 39999], x[-2, 1] = 3.0, 2.0
    tokens = torch.full((x.shape[0],), 39999, device="cuda")
    lp, ent, tl, ti = gpu.token_logprobs_dev(x, tokens, top=1)
    assert ti[-1].item() == 39999 and ti[-2].item() == 1 and ti[0].item() == 0
    assert abs(lp[-1].item() - (3 - math.log(39999 + math.exp(3)))) < 1e-5


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_rows_whose_best_come_late(gpu, dtype):
    """Rows that rise towards their end: bounds that are found while other warps go on must never pass the alternatives that are wanted."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(1500, 9001, generator=g) + torch.arange(9001)[None] * (torch.rand(1500, 1, generator=g) * 1e-3)
    check(gpu, x.to(DT[dtype]).cuda(), torch.randint(9001, (1500,), generator=g).cuda(), 10)
