"""Rotary positions on the GPU against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import plain_kv4 as plain

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def bound(x, want, dtype):
    """f32: 2^-23 of the result, and 2^-46 of the pair (what two f32 leave of a sine); 16-bit types: 2^-21 of the largest element, four roundings to f32 of it, and the result's own."""
    top = np.abs(x).max(initial=0.0) * 2
    if dtype == "float32":
        return np.abs(want) * 2.0 ** -22 + top * 2.0 ** -45 + 2.0 ** -148
    return np.abs(want) * (plain.EPS[dtype] + 2.0 ** -22) + top * 2.0 ** -21 + plain.TINY[dtype]


def table(gpu, rot, theta=10000.0):
    t = gpu.rope_turns(theta, rot)
    return t, torch.from_numpy(t.view("int64")).cuda()


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,heads,dim,rot", [(1, 32, 64, 64), (1, 1, 128, 128), (7, 5, 128, 96), (300, 3, 80, 64), (3, 2, 1, 0), (5, 3, 33, 18), (9, 4, 256, 2), (1200, 2, 64, 32), (2, 1, 1024, 1024), (6, 70, 16, 16)])
def test_rope(gpu, rows, heads, dim, rot, layout, dtype):
    rng = np.random.default_rng(rows + dim)
    x = torch.from_numpy(rng.normal(0, 1, (rows, heads, dim)).astype(np.float32)).to(DT[dtype])
    y = torch.from_numpy(rng.normal(0, 1, (rows, 2, dim)).astype(np.float32)).to(DT[dtype])
    pos = rng.integers(0, 2 ** 20, rows)
    pos[0] = 0 if rows > 1 else 131_071
    turns, on_gpu = table(gpu, rot)
    on_pos = torch.from_numpy(pos).cuda()
    for inverse, magnitude in ((False, 1.0), (True, 1.3)):
        out, y_out = gpu.rope_dev(x.cuda(), on_pos, on_gpu, layout=layout, inverse=inverse, magnitude=magnitude, y=y.cuda())
        for a, b in ((x, out), (y, y_out)):
            a64 = a.double().numpy()
            want = plain.rotate(a64, turns, pos, layout, magnitude, inverse)
            assert (np.abs(b.double().cpu().numpy() - want) <= bound(a64, want, dtype)).all()
    alone = gpu.rope_dev(x.cuda(), on_pos, on_gpu, layout=layout, inverse=True, magnitude=1.3)
    assert (alone == out).all()


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("pad,dim,rot", [(0, 64, 64), (8, 64, 48), (3, 64, 64), (1, 40, 20)])
def test_in_place_and_strided(gpu, pad, dim, rot, layout, dtype):
    rows, heads = 37, 6
    rng = np.random.default_rng(dim + pad)
    wide = torch.from_numpy(rng.normal(0, 1, (rows, heads * dim + pad)).astype(np.float32)).to(DT[dtype]).cuda()
    before = wide.clone()
    x = wide[:, pad:].unflatten(1, (heads, dim))
    turns, on_gpu = table(gpu, rot)
    pos = torch.arange(1000, 1000 + rows).cuda()
    fresh = gpu.rope_dev(x, pos, on_gpu, layout=layout)
    assert gpu.rope_dev(x, pos, on_gpu, layout=layout, out=x) is x
    assert (x == fresh).all() and (wide[:, :pad] == before[:, :pad]).all()
    want = plain.rotate(before[:, pad:].unflatten(1, (heads, dim)).double().cpu().numpy(), turns, pos.tolist(), layout)
    assert (np.abs(x.double().cpu().numpy() - want) <= bound(want, want, dtype)).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_is_the_turn_back(gpu, layout):
    """For a loss sum(g * rope(x)) the gradient is the inverse turn of g: against differences in each element."""
    rng = np.random.default_rng(1)
    rows, heads, dim, rot = 4, 2, 32, 24
    x, g = (torch.from_numpy(rng.normal(0, 1, (rows, heads, dim)).astype(np.float32)).cuda() for _ in range(2))
    turns, on_gpu = table(gpu, rot)
    pos = torch.tensor([0, 3, 77, 5000]).cuda()
    call = lambda t, inverse=False: gpu.rope_dev(t, pos, on_gpu, layout=layout, magnitude=1.1, inverse=inverse)  # noqa: E731
    grad = call(g, True)
    for d in range(dim):
        step = torch.zeros_like(x)
        step[..., d] = 1.0
        # linear: a step of 1 in one element of every head changes that head's loss by its gradient, up to f32's rounding of 32 terms of size 4
        diff = ((call(x + step).double() - call(x).double()) * g.double()).sum(-1)
        assert (diff - grad[..., d].double()).abs().max() < 32 * 4 * 2.0 ** -22
    back = call(call(x), True) / 1.21
    assert (back[..., :rot] - x[..., :rot]).abs().max() < 2.0 ** -20


def test_far_positions_and_wrapping(gpu):
    """Positions past 2^32 and below 0 lose nothing."""
    x = torch.randn(5, 2, 64, device="cuda")
    turns, on_gpu = table(gpu, 64)
    pos = torch.tensor([2 ** 33 + 5, 2 ** 62, -1, -10 ** 12, 2 ** 63 - 1]).cuda()
    got = gpu.rope_dev(x, pos, on_gpu)
    want = plain.rotate(x.double().cpu().numpy(), turns, pos.tolist())
    assert (np.abs(got.double().cpu().numpy() - want) <= bound(x.double().cpu().numpy(), want, "float32")).all()


def test_captured_and_on_other_streams(gpu):
    x, pos = torch.randn(9, 4, 128, device="cuda"), torch.arange(9).cuda()
    _, on_gpu = table(gpu, 128)
    out = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.rope_dev(x, pos, on_gpu, out=out)
    pos += 100
    graph.replay()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    other = gpu.rope_dev(x, pos, on_gpu, stream=stream)
    torch.cuda.synchronize()
    assert (out == other).all() and (out[1:] != x[1:]).any()


@pytest.mark.parametrize("heads,dim,rot", [(3001, 33, 18), (2500, 32, 16)])
def test_many_heads(gpu, heads, dim, rot):
    x = torch.randn(5, heads, dim, device="cuda")
    turns, on_gpu = table(gpu, rot)
    pos = torch.arange(5).cuda() * 1000
    got = gpu.rope_dev(x, pos, on_gpu)
    x64 = x.double().cpu().numpy()
    want = plain.rotate(x64, turns, pos.tolist())
    assert (np.abs(got.double().cpu().numpy() - want) <= bound(x64, want, "float32")).all()


def test_refusals(gpu):
    x, pos = torch.randn(3, 2, 64, device="cuda"), torch.arange(3).cuda()
    _, on_gpu = table(gpu, 64)
    for call in (lambda: gpu.rope_dev(x, pos[:2], on_gpu), lambda: gpu.rope_dev(x, pos.int(), on_gpu), lambda: gpu.rope_dev(x.double(), pos, on_gpu), lambda: gpu.rope_dev(x[..., ::2], pos, on_gpu),
                 lambda: gpu.rope_dev(x, pos, on_gpu.double()), lambda: gpu.rope_dev(x, pos, on_gpu, layout="other"), lambda: gpu.rope_dev(x, pos.cpu(), on_gpu),
                 lambda: gpu.rope_dev(x, pos, on_gpu, y=x.half()), lambda: gpu.rope_dev(x, pos, on_gpu, out=x[:2])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(gpu.LeafcutterError):
        gpu.rope_dev(x[..., :32].contiguous(), pos, on_gpu)   # more dims turned than there are
    assert gpu.rope_dev(x[:0], pos[:0], on_gpu).shape == (0, 2, 64)
