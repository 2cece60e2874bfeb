"""Calls over the 4-bit cache that its documentation allows at its ends: groups that do not divide a tile, as many sequences as there may be, rows in any order, windows at every border of a tile,
scales of 0, queries as they were at the time of the call, several streams at once."""
import math

import numpy as np
import pytest
import torch

import plain_kv4 as plain
from test_kv4_gpu import DT, Setup, check_attention, cuda, host, mass_bound

pytestmark = pytest.mark.gpu


def weigh(s, q, q64, wlse, big, weights, window=0):
    mass = torch.zeros(len(s.seqs), s.kv, s.table.shape[1] * s.page, device="cuda")
    s.cache.weights(s.batch, q, cuda(wlse.astype(np.float32)), mass, window=window)
    want = np.zeros(mass.shape)
    group = q64.shape[1] // s.kv
    for i, r, h, lo, p in weights:
        want[i, h // group, lo:lo + len(p)] += p
    bound = mass_bound(want, weights, plain.score_bound(big, s.dim), group, want.shape, np.abs(wlse) * 2.0 ** -23)
    assert (np.abs(host(mass) - want) <= bound).all()


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("kv,heads,dim,seqs", [(1, 12, 64, [(40, 30), (300, 23)]), (4, 12, 96, [(10, 100)]), (1, 7, 128, [(0, 40), (250, 1), (100, 19)]), (2, 2, 112, [(500, 140)]), (1, 5, 256, [(30, 60)]),
                                               (1, 40, 32, [(129, 7), (0, 4)])], ids=str)
def test_groups_of_any_size(gpu, kv, heads, dim, seqs, dtype):
    s = Setup(gpu, seqs, kv, dim, 16, seed=dim)
    q, q64 = s.normal(heads, dtype)
    out, lse = torch.empty_like(q), torch.empty(s.rows, heads, device="cuda")
    s.cache.attention(s.batch, q, out, lse=lse)
    weights = check_attention(s, out, lse, q64, dtype)
    _, wlse, _, big, _, _ = s.plain.attention(s.table, s.ctx, s.start, q64)
    weigh(s, q, q64, wlse, big, weights)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [127, 128, 129, 255, 256, 257, 400])
def test_windows_at_the_borders_of_tiles(gpu, window, dtype):
    s = Setup(gpu, [(385, 130), (0, 258)], 1, 64, 32, seed=window)
    q, q64 = s.normal(2, dtype)
    out, lse = torch.empty_like(q), torch.empty(s.rows, 2, device="cuda")
    s.cache.attention(s.batch, q, out, lse=lse, window=window)
    weights = check_attention(s, out, lse, q64, dtype, None, window)
    _, wlse, _, big, _, _ = s.plain.attention(s.table, s.ctx, s.start, q64, None, window)
    weigh(s, q, q64, wlse, big, weights, window)


@pytest.mark.parametrize("rows", [1, 130])
def test_pages_in_front_of_windows_are_not_looked_at(gpu, rows):
    s = Setup(gpu, [(700, rows)], 2, 64, 16, seed=1)
    q, q64 = s.normal(4, "bfloat16")
    window = 100
    table = s.table.copy()
    table[0, :(700 - window + 1) // 16] = 10 ** 9
    batch = s.rows_of(rows, table=table)
    out, lse = torch.empty_like(q), torch.empty(rows, 4, device="cuda")
    s.cache.attention(batch, q, out, lse=lse, window=window)
    check_attention(s, out, lse, q64, "bfloat16", None, window)
    mass = torch.zeros(1, 2, s.table.shape[1] * 16, device="cuda")
    s.cache.weights(batch, q, lse, mass, window=window)
    assert s.status.item() == 0 and abs(mass.sum().item() - 4 * rows) < 0.01 * rows


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_as_many_sequences_as_there_may_be(gpu, dtype):
    n, kv, dim, page = 4096, 1, 32, 16
    rng = np.random.default_rng(0)
    seqs = [(int(c), 0 if i % 5 == 3 else 1) for i, c in enumerate(rng.integers(0, 40, n))]
    s = Setup(gpu, seqs, kv, dim, page, seed=2)
    q, q64 = s.normal(2, dtype)
    out, lse = torch.empty_like(q), torch.empty(s.rows, 2, device="cuda")
    for hint in (1, 100):                                                   # by either kernel
        s.cache.attention(s.rows_of(hint), q, out, lse=lse)
        weights = check_attention(s, out, lse, q64, dtype)
        mass = torch.zeros(n, kv, 48, device="cuda")
        s.cache.weights(s.rows_of(hint * 3), q, lse, mass)
        want = np.zeros((n, kv, 48))
        for i, r, h, lo, p in weights:
            want[i, 0, lo:lo + len(p)] += p
        assert np.abs(host(mass) - want).max() < 2e-5
    kept, ctx = s.cache.evict(s.batch, mass, 20, recent=2)
    for i in (0, 1, 2, 3, 77, 4095):
        stays = plain.evict(host(mass)[i, 0] if sum(seqs[i]) <= 20 else want[i, 0].astype(np.float32), sum(seqs[i]), 20, 20, 2, 0)
        assert ctx[i].item() == min(20, sum(seqs[i])) and (sum(seqs[i]) <= 20 or len(stays) == 20)
        assert (kept[i, 0, :min(20, sum(seqs[i]))] >= 0).all() and (kept[i, 0, min(20, sum(seqs[i])):] == -1).all()


def test_sequences_in_any_order_and_rows_of_none(gpu):
    """row_start that goes back and forth over rows that no two sequences share."""
    s = Setup(gpu, [(20, 3), (9, 0), (40, 2)], 2, 64, 16, seed=5)
    (k, k64), (q, q64) = s.normal(2, "bfloat16"), s.normal(4, "bfloat16")
    start = np.array([2, 5, 0, 2], np.int32)                               # sequence 0: rows 2-4; 1: broken; 2: rows 0-1
    batch = s.rows_of(3, start=start)
    s.cache.append(batch, k, k)
    assert s.status.item() == 2
    order = [(0, 2, 3), (2, 0, 2)]
    for i, r0, n in order:
        s.plain.append(s.table[i:i + 1], s.ctx[i:i + 1], np.array([r0, r0 + n]), k64, k64, [])
    s.check_pools()
    out, lse = torch.zeros_like(q), torch.zeros(s.rows, 4, device="cuda")
    s.cache.attention(batch, q, out, lse=lse)
    for i, r0, n in order:
        want = s.plain.attention(s.table[i:i + 1], s.ctx[i:i + 1], np.array([0, n]), q64[r0:r0 + n])[0]
        assert np.abs(host(out)[r0:r0 + n] - want).max() < 0.02


def test_scales_of_nothing(gpu):
    """A head whose scale is 0 holds zeros; attention over zeros is their mean."""
    s = Setup(gpu, [(0, 20)], 2, 32, 16, seed=6)
    for t, a in ((s.pools[4], s.plain.k_scale), (s.pools[5], s.plain.v_scale)):
        t[1] = 0.0
        a[1] = 0.0
    k, k64 = s.normal(2, "float32")
    q, q64 = s.normal(2, "float32")
    s.cache.append(s.batch, k, k)
    back = torch.empty_like(k)
    s.cache.read(s.batch, back, None)
    assert (back[:, 1] == 0).all() and (s.pools[0][cuda(s.table[0].astype(np.int64)), 1, :4] == 0x88).all()
    out, lse = torch.empty_like(q), torch.empty(20, 2, device="cuda")
    s.cache.attention(s.batch, q, out, lse=lse)
    assert (out[:, 1] == 0).all() and np.abs(host(lse)[:, 1] - np.log(np.arange(1, 21))).max() < 1e-6


def test_calls_on_two_streams_at_once(gpu):
    """Attention by tiles and weights by tiles, which share an SM's tensor memory, and eviction, on streams of their own."""
    kv, heads, dim = 4, 16, 128
    s = Setup(gpu, [(900, 100), (300, 64)], kv, dim, 16, seed=7)
    q, q64 = s.normal(heads, "bfloat16")
    lse = torch.empty(s.rows, heads, device="cuda")
    first = s.cache.attention(s.batch, q, lse=lse)
    mass0 = torch.rand(2, kv, 1024, device="cuda")
    mass1 = s.cache.weights(s.batch, q, lse, mass0.clone())
    other = Setup(gpu, [(2000, 0), (1500, 1)], kv, dim, 16, seed=8)
    sums = torch.rand(2, kv, 2048, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(3)]
    ws = torch.empty(s.cache.attention_workspace(s.batch, q), dtype=torch.uint8, device="cuda")
    outs, masses, kept = [torch.empty_like(q) for _ in range(10)], [mass0.clone() for _ in range(10)], []
    torch.cuda.synchronize()
    for i in range(10):
        s.cache.attention(s.batch, q, outs[i], workspace=ws, stream=streams[0])
        s.cache.weights(s.batch, q, lse, masses[i], stream=streams[1])
        kept.append(other.cache.evict(other.batch, sums.clone(), 500, stream=streams[2])[0])
        torch.cuda.synchronize()
    assert all((o == first).all() for o in outs) and all((m == mass1).all() for m in masses) and all((k == kept[0]).all() for k in kept)


def test_a_first_call_inside_a_capture(gpu):
    """Kernels that nothing has launched before, captured."""
    s = Setup(gpu, [(10, 70)], 1, 80, 16, seed=9)
    q, q64 = s.normal(3, "float16")
    out, lse, mass = torch.empty_like(q), torch.empty(s.rows, 3, device="cuda"), torch.zeros(1, 1, 80, device="cuda")
    kept, ctx = torch.empty(1, 1, 40, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(s.cache.attention_workspace(s.batch, q), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.cache.attention(s.batch, q, out, lse=lse, workspace=ws)
        s.cache.weights(s.batch, q, lse, mass)
        s.cache.evict(s.batch, mass, 40, kept=kept, ctx_out=ctx)
    graph.replay()
    torch.cuda.synchronize()
    check_attention(s, out, lse, q64, "float16")
    assert ctx.item() == 40 and abs(mass.sum().item()) <= 210.1 and (kept[0, 0].diff() > 0).all()


def test_a_smaller_workspace_is_refused(gpu):
    s = Setup(gpu, [(100, 1)], 2, 64, 16)
    q, _ = s.normal(4, "bfloat16")
    need = s.cache.attention_workspace(s.batch, q)
    with pytest.raises(gpu.LeafcutterError):
        s.cache.attention(s.batch, q, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    assert need > 16
    with pytest.raises(gpu.LeafcutterError):
        s.cache.evict(s.batch, torch.zeros(2, 2, 200, device="cuda")[:1], 10, ctx_out=s.batch._kept[1])   # the lengths that are still read
    for bad in (dict(lse=torch.empty(1, 4)), dict(lse=torch.empty(1, 3, device="cuda")), dict(out=torch.empty(1, 4, 32, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(ValueError):
            s.cache.attention(s.batch, q, **bad)
    with pytest.raises(ValueError):
        s.cache.weights(s.batch, q, torch.empty(1, 4, device="cuda"), torch.zeros(1, 3, 200, device="cuda"))
    with pytest.raises(ValueError):
        s.cache.weights(s.batch, q, torch.empty(1, 4, device="cuda"), torch.zeros(1, 2, 400, device="cuda")[..., ::2])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("seqs", [[(300, 1), (40, 1)], [(30, 21)], [(200, 160)]], ids=["few", "some", "many"])
def test_rows_of_zeros_beside_queries_that_only_a_large_scale_brings_back(gpu, seqs, dtype):
    """A scale of 2^126 for queries of 2^-130: a row of zeros, and the rows that fill up a tile, have scores of 0 all the same."""
    s = Setup(gpu, seqs, 1, 128, 16, seed=4)
    s.pools[4].fill_(1.0)
    s.plain.k_scale[:] = 1.0
    q = s.normal(4, "float32")[0].mul_(2.0 ** -130).to(DT[dtype])
    q[:, 2] = 0.0
    q64 = q.double().cpu().numpy()
    out, lse = torch.empty_like(q), torch.empty(s.rows, 4, device="cuda")
    s.cache.attention(s.batch, q, out, lse=lse, scale=2.0 ** 126)
    weights = check_attention(s, out, lse, q64, dtype, 2.0 ** 126)
    _, wlse, _, big, _, _ = s.plain.attention(s.table, s.ctx, s.start, q64, 2.0 ** 126)
    mass = torch.zeros(len(seqs), 1, s.table.shape[1] * s.page, device="cuda")
    s.cache.weights(s.batch, q, cuda(wlse.astype(np.float32)), mass, scale=2.0 ** 126)
    want = np.zeros(mass.shape)
    for i, r, h, lo, p in weights:
        want[i, 0, lo:lo + len(p)] += p
    bound = mass_bound(want, weights, plain.score_bound(big, s.dim), 4, want.shape, np.abs(wlse) * 2.0 ** -23)
    assert (np.abs(host(mass) - want) <= bound).all()


@pytest.mark.parametrize("ties", ["none", "many", "odd"])
@pytest.mark.parametrize("length,keep,off", [(259_065, 100_003, 0), (259_072, 17, 1), (70_001, 70_000, 0), (130_000, 64_999, 3)])
def test_evict_of_as_long_contexts_as_clusters_hold(gpu, length, keep, off, ties):
    """Blocks of up to 32,384 sums, at any alignment; shorter sequences in the same tables."""
    page, pages = 16, -(-length // 16)
    rng = np.random.default_rng(length)
    table = rng.permutation(pages + 3000).astype(np.int32)[:pages]
    tables = np.full((2, pages), -1, np.int32)
    tables[0] = table
    rest = np.setdiff1d(np.arange(pages + 3000), table)[:2000]
    tables[1, :2000] = rest
    lengths = [length, 31_990]
    pools = [rng.integers(0, 256, (pages + 3000, 1, page, n)).astype(np.uint8) for n in (8, 8, 1, 1)]
    on_gpu = [cuda(a) for a in pools]
    cache = gpu.Kv4Cache(*on_gpu, torch.ones(1, device="cuda"), torch.ones(1, device="cuda"))
    rows = gpu.Kv8Rows(cuda(tables), cuda(np.array(lengths, np.int32)), cuda(np.zeros(3, np.int32)), 0)
    mass = rng.lognormal(0, 2, (2, 1, page * pages + 4)).astype(np.float32)
    if ties == "many":
        mass = np.floor(np.minimum(mass, 3.0))
    elif ties == "odd":
        mass = np.where(rng.random(mass.shape) < 0.3, rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0, 1e-45], np.float32), mass.shape), mass).astype(np.float32)
    whole = cuda(mass)
    kept, ctx = cache.evict(rows, whole[:, :, off:off + page * pages], keep, recent=5, first=3)
    want, pool_want = mass.copy(), [p.copy() for p in pools]
    for i, n in enumerate(lengths):
        m, got = mass[i, 0, off:off + n], kept[i, 0].cpu().numpy()
        if n <= keep:
            assert ctx[i].item() == n and (got[:n] == np.arange(n)).all() and (got[n:] == -1).all()
            continue
        inner = np.arange(3, n - 5)
        nan = np.isnan(m[inner])
        order = inner[np.lexsort((inner, -np.where(nan, 0.0, m[inner]), nan))][:keep - 8]   # NaN last, then the larger, then the lower slot
        stays = np.sort(np.concatenate((np.arange(3), order, np.arange(n - 5, n))))
        assert ctx[i].item() == keep and (got == stays).all()
        want[i, 0, off:off + n] = 0.0
        want[i, 0, off:off + keep] = m[stays]
        for p, old in zip(pool_want, pools):
            p[tables[i][np.arange(keep) // page], 0, np.arange(keep) % page] = old[tables[i][stays // page], 0, stays % page]
    assert np.array_equal(host(whole), want, equal_nan=True)
    for t, p in zip(on_gpu, pool_want):
        assert (t.cpu().numpy() == p).all()
