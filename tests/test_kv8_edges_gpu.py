"""The 8-bit key/value cache on the GPU at the edges of what its calls allow: workspaces that serve smaller calls, tables far wider than contexts, windows whose
pages are gone, rows of very different size, numbers that are not finite, values next to zero, bad pages in the middle of a draft."""
import math

import numpy as np
import pytest
import torch

import plain_kv8 as plain
from test_kv8_gpu import DT, Setup, check_attention, cuda, host

pytestmark = pytest.mark.gpu


def check_relative(s, heads, dtype, q):
    """As check_attention, for weights and values of any size: what a weight loses below f16's normal range counts against the row's largest weight and the
    largest value scale, not against 1 or the output."""
    q, q64 = q
    out = torch.full_like(q, math.nan)
    s.cache.attention(s.batch, q, out)
    want, mass, big, keys = s.plain.attention(s.table, s.ctx, s.start, q64)
    split = dtype == "float32"
    d = big * (2.0 ** -22 + (s.dim / 16 + 4) * 2.0 ** -23) + 2.0 ** -21
    eps = 2 * (d[..., None] + (2.0 ** -22 if split else 2.0 ** -11)) + 2.0 ** -20
    # a weight below 2^-14 (f32: its low part) is off by 2^-25 at most, values are 127 of their scale, and the sum of weights is 2^6 or more;
    # the last term is the rounding of numbers below the types' normal range
    low = 2.0 ** -31 * keys[:, None, None] * 127 * s.plain.v_scale.max()
    bound = mass * eps + low + np.abs(want) * (plain.EPS[dtype] / 2 + 2.0 ** -23) + (2.0 ** -149 if split else max(plain.TINY[dtype], 2.0 ** -134))
    err = np.abs(host(out).astype(np.float64) - want)
    assert (err <= bound).all(), f"{np.nanmax(err / np.maximum(bound, 1e-300)):.2f} of the bound"
    assert s.status.item() == 0
    assert np.abs(want).max() > 100 * low.max() or not split
    return out


def want_of(s, heads, q64, dtype, window=0):
    want, mass, big, keys = s.plain.attention(s.table, s.ctx, s.start, q64, None, window)
    return want, plain.attention_bound(want, mass, big, keys, s.dim, dtype, dtype == "float32")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (8, 2, 64), (4, 1, 256)])
def test_a_workspace_serves_smaller_calls(gpu, dtype, heads, kv, dim):
    """One workspace, asked for with the largest chunk, for shorter chunks and single tokens after it."""
    pages = 2
    pools = [torch.randint(-127, 128, (pages, kv, 16, dim), dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.full((pages, kv), 0.01, device="cuda") for _ in range(2)]
    cache = gpu.Kv8Cache(*pools)
    table = torch.zeros(4, 512, dtype=torch.int32, device="cuda")       # 8,192 positions, all on one page
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    largest = 4096
    q = torch.randn(largest, heads, dim, device="cuda").to(DT[dtype])
    ws = torch.empty(cache.attention_workspace(gpu.Kv8Rows(table, i32([0] * 4), i32([0] * 5), largest), q), dtype=torch.uint8, device="cuda")
    for n in (4096, 2048, 1024, 512, 256, 64, 33, 8, 1):
        for seqs in (1, 4):
            for max_rows in sorted({n, 1, -(-n // seqs)}):
                start = [n * i // seqs for i in range(seqs + 1)]
                rows = gpu.Kv8Rows(table[:seqs], i32([5] * seqs), i32(start), max_rows)
                assert cache.attention_workspace(rows, q[:n]) <= ws.numel()
                out = cache.attention(rows, q[:n], workspace=ws)
                if n <= 64:
                    assert torch.equal(out, cache.attention(rows, q[:n]))
    torch.cuda.synchronize()


def test_workspaces_grow_with_their_calls(gpu):
    """Whatever a call has less of than another, its workspace is no larger."""
    rng = np.random.default_rng(21)
    pools = [torch.zeros(1, 8, 16, 128, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.zeros(1, 8, device="cuda") for _ in range(2)]
    cache = gpu.Kv8Cache(*pools)
    z = torch.zeros(1, dtype=torch.int32, device="cuda").data_ptr()
    import ctypes as C

    def size(typ, n_seqs, width, max_rows, n_rows, heads):
        rows, out = gpu._capi.Kv8RowsStruct(z, z, z, None, n_seqs, width, max_rows, 0), C.c_size_t()
        gpu._capi.check(gpu.load().lc_attention_kv8_workspace(cache._ref, C.byref(rows), typ, n_rows, heads, C.byref(out)))
        return out.value
    for _ in range(300):
        typ, heads = int(rng.choice([0, 1, 30])), int(rng.choice([8, 16, 32, 64]))
        big = [int(np.exp(rng.uniform(0, math.log(m)))) for m in (256, 4096, 4096, 8192)]
        small = [int(rng.integers(0, b + 1)) for b in big]
        assert size(typ, *small, heads) <= size(typ, *big, heads), (typ, heads, small, big)


@pytest.mark.parametrize("dtype,heads,kv,dim,new,max_rows", [("bfloat16", 64, 8, 128, 4096, 4096), ("float32", 64, 8, 128, 4096, 4096), ("bfloat16", 64, 8, 128, 4096, 1), ("bfloat16", 16, 8, 64, 3, 3),
                                                             ("bfloat16", 64, 8, 256, 6000, 6000)])
def test_tables_for_a_million_positions(gpu, dtype, heads, kv, dim, new, max_rows):
    """A table far wider than the contexts: the same results as with a narrow one."""
    pages = -(-(new + 20) // 16)
    pools = [torch.randint(-127, 128, (pages, kv, 16, dim), dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.rand(pages, kv, device="cuda") * 0.02 for _ in range(2)]
    cache = gpu.Kv8Cache(*pools)
    wide = torch.full((1, 2 ** 16), -1, dtype=torch.int32, device="cuda")
    wide[0, :pages] = torch.randperm(pages, device="cuda").to(torch.int32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(new, heads, dim, device="cuda").to(DT[dtype])
    outs = []
    for table in (wide, wide[:, :pages].contiguous()):
        status = i32([0])
        rows = gpu.Kv8Rows(table, i32([20]), i32([0, new]), max_rows, status)
        outs.append(cache.attention(rows, q).double())
        assert status.item() == 0
    # both are sums of the same terms, in f32 and in another order at most; then one rounding each
    assert (outs[0] - outs[1]).abs().max() <= outs[1].abs().max() * (plain.EPS[dtype] + 2.0 ** -10 * (dtype != "float32") + 2.0 ** -18)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("seqs,window", [([(1000, 40), (700, 64), (333, 33), (1001, 150)], 100), ([(300, 70), (129, 130), (200, 64), (77, 40)], 37), ([(1000, 3), (500, 1), (777, 2)], 100)])
def test_pages_in_front_of_a_window_are_gone(gpu, dtype, page, seqs, window):
    """A serving loop drops the pages that no row sees any more, and their numbers, or what stands there, mean nothing."""
    s = Setup(gpu, seqs, 4, 64, page, seed=31)
    q = s.normal(16, dtype)
    first = check_attention(s, 16, dtype, window=window, q=q).clone()
    gone = [(i, p) for i, (c, _) in enumerate(seqs) for p in range(s.table.shape[1]) if (p + 1) * page <= c - window + 1]
    assert gone
    for scale, bad in zip(s.pools[2:], (math.nan, math.inf)):
        for i, p in gone:
            scale[int(s.table[i, p])] = bad
    assert torch.equal(first, check_attention(s, 16, dtype, window=window, q=q))
    table = s.table.copy()
    for number in (-1, 2 ** 31 - 1):
        for i, p in gone:
            table[i, p] = number
        s.batch = s.rows_of(max(n for _, n in seqs), table=table)
        assert torch.equal(first, check_attention(s, 16, dtype, window=window, q=q))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("q_scale", [1e4, 1e8, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("seqs,heads", [([(300, 100), (0, 130), (64, 70)], 8), ([(300, 2), (5000, 1)], 8), ([(3000, 90)], 16)])
def test_scores_far_beyond_softmaxs_range(gpu, dtype, q_scale, seqs, heads):
    """One key has all of the weight: where the best two scores differ by more than their errors, the output is its value."""
    s = Setup(gpu, seqs, 4, 64, 16, seed=35)
    q, q64 = s.normal(heads, dtype, q_scale)
    out = host(check_relative(s, heads, dtype, (q, q64))).astype(np.float64)
    n_clear = 0
    for i, (c, n) in enumerate(s.seqs):
        k, v = s.plain.values("k", s.table[i], c + n), s.plain.values("v", s.table[i], c + n)
        for j in range(n):
            r = int(s.start[i]) + j
            for h in range(heads):
                g = h // (heads // 4)
                score = k[:c + j + 1, g] @ q64[r, h] / 8
                best = int(score.argmax())
                # a score is off by 2^-17 of the sum of its terms' magnitudes at most (queries in 22 bits, 8 additions cut off, roundings); 40: weights below e^-40
                if (score[best] - np.delete(score, best)).min(initial=np.inf) < 2.0 ** -16 * (np.abs(k[:c + j + 1, g]) @ np.abs(q64[r, h]) / 8).max() + 40:
                    continue
                n_clear += 1
                # the value is an integer times two roundings' scale, its weight over itself rounded to 11 bits, then the output's rounding
                assert (np.abs(out[r, h] - v[best, g]) <= np.abs(v[best, g]) * (plain.EPS[dtype] / 2 + 2.0 ** -20 + (dtype != "float32") * 2.0 ** -10) + 1e-12).all(), (r, h)
    assert n_clear > s.rows * heads / 2


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,kv,dim,seqs", [(8, 4, 128, [(300, 100), (0, 130), (64, 70)]), (8, 8, 64, [(600, 200), (33, 129)]), (12, 4, 96, [(40, 90)] * 3)])
def test_rows_of_very_different_size_side_by_side(gpu, dtype, heads, kv, dim, seqs):
    """What a row gives does not depend on how large the others of its call are."""
    s = Setup(gpu, seqs, kv, dim, 16, seed=41)
    q, q64 = s.normal(heads, dtype)
    alone = check_attention(s, heads, dtype, q=(q, q64)).clone()
    large = s.rng.random(s.rows) < 0.5
    up = 2.0 ** 12 if dtype == "float16" else 2.0 ** 40                 # exact in every type
    q64 = q64 * np.where(large, up, 1.0)[:, None, None]
    q = torch.from_numpy(q64).to(DT[dtype]).cuda()
    assert np.array_equal(q.double().cpu().numpy(), q64)
    both = check_relative(s, heads, dtype, (q, q64))
    assert torch.equal(both[~large], alone[~large])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("sizes", [(-12, 12), (-25, -5)])
def test_rows_of_all_sizes(gpu, dtype, sizes):
    s = Setup(gpu, [(200, 128), (70, 80)], 4, 64, 16, seed=42)
    q64 = s.rng.normal(0, 1, (s.rows, 16, 64)) * 10.0 ** s.rng.uniform(*sizes, (s.rows, 16, 1))
    q = torch.from_numpy(q64).to(DT[dtype])
    check_relative(s, 16, dtype, (q.cuda(), q.double().numpy()))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,kv,seqs", [(16, 4, [(0, 130), (5, 70), (300, 64)]), (4, 4, [(0, 3), (40, 1), (700, 4)])])
def test_rows_that_are_not_finite(gpu, dtype, heads, kv, seqs):
    """A row with an infinity or NaN is NaN, the first one of a prompt, which sees one key, among them; the others are as ever."""
    s = Setup(gpu, seqs, kv, 64, 16, seed=51)
    s.plain.k[..., 3] = np.where(s.plain.k[..., 3] == 0, -5, -np.abs(s.plain.k[..., 3]))   # one sign: an infinity alone gives scores of minus infinity
    s.pools[0].copy_(torch.from_numpy(s.plain.k))
    q, q64 = s.normal(heads, dtype)
    bad = {}
    for i, (at, n) in enumerate(zip(s.start, np.diff(s.start))):
        for j, x in enumerate((math.inf, -math.inf, math.nan)):
            if j < n:
                bad[int(at) + (j if i != 1 else n - 1 - j)] = (x, (i + j) % heads)
    for r, (x, h) in bad.items():
        q[r, h, 3] = x
        q64[r, h] = 0.0
    out = torch.zeros_like(q)
    s.cache.attention(s.batch, q, out)
    want, bound = want_of(s, heads, q64, dtype)
    out = host(out).astype(np.float64)
    nan = np.zeros(out.shape[:2], bool)
    for r, (x, h) in bad.items():
        nan[r, h] = True
    assert np.isnan(out[nan]).all()
    assert (np.abs(out - want)[~nan] <= bound[~nan]).all()
    assert s.status.item() == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("where", ["first", "middle", "last", "all but one"])
@pytest.mark.parametrize("exponent", [0, -16, -40, -110, -130])
@pytest.mark.parametrize("page", [16, 128])
def test_tiles_of_values_that_are_zero(gpu, dtype, where, exponent, page):
    """128 keys whose values have scale 0 count in the denominator alone, however small the scales of the others are."""
    s = Setup(gpu, [(520, 70), (384, 128), (700, 64)], 4, 64, page, seed=61)
    s.plain.v_scale *= np.float32(2.0) ** np.float32(exponent / 2)      # in two steps: the power itself may be below the smallest number
    s.plain.v_scale *= np.float32(2.0) ** np.float32(exponent / 2)
    per = 128 // page
    for i, (c, n) in enumerate(s.seqs):
        tiles = -(-(c + n) // 128)
        zero = {"first": [0], "middle": [tiles // 2], "last": [tiles - 1], "all but one": [t for t in range(tiles) if t != 2]}[where]
        for t in zero:
            for p in s.table[i, t * per:(t + 1) * per]:
                if p >= 0:
                    s.plain.v_scale[p] = 0.0
    s.pools[3].copy_(torch.from_numpy(s.plain.v_scale))
    check_relative(s, 16, dtype, s.normal(16, dtype))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("small", [2.0 ** -50, 1e-39, 1e-44])
def test_a_page_of_values_next_to_nothing(gpu, dtype, small):
    """One page whose values are all but zero, among others: as good as zeros, for every row."""
    s = Setup(gpu, [(520, 70), (384, 128), (700, 64), (5, 1)], 4, 64, 16, seed=62)
    for i, p in ((0, 3), (1, 0), (2, 40)):
        s.plain.v_scale[s.table[i, p]] = small
    s.pools[3].copy_(torch.from_numpy(s.plain.v_scale))
    check_relative(s, 16, dtype, s.normal(16, dtype))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,kv,new", [(4, 2, 5), (4, 4, 20), (1, 1, 2), (16, 4, 80)])
@pytest.mark.parametrize("window", [0, 9])
def test_rows_that_do_not_need_a_bad_page(gpu, dtype, heads, kv, new, window):
    """A page outside the pool makes NaN of the rows that see a position of it; rows in front of it, and those whose window has left it, are as ever."""
    seqs = [(46, new), (300, new), (17, new)]
    for i, page in ((0, 3), (1, 300 // 16), (1, (300 + new - 1) // 16), (2, 1)):
        s = Setup(gpu, seqs, kv, 64, 16, seed=71)
        q, q64 = s.normal(heads, dtype)
        want, bound = want_of(s, heads, q64, dtype, window)
        table = s.table.copy()
        table[i, page] = (-1, 10 ** 6)[page % 2]
        out = torch.full_like(q, 7.0)
        s.cache.attention(s.rows_of(new, table=table), q, out, window=window)
        out = host(out).astype(np.float64)
        bad = np.zeros(s.rows, bool)
        for j in range(new):
            pos = seqs[i][0] + j
            bad[s.start[i] + j] = page * 16 <= pos and (not window or page * 16 + 15 > pos - window)
        assert np.isnan(out[bad]).all()
        assert (np.abs(out - want)[~bad] <= bound[~bad]).all()
        assert s.status.item() == (i + 1 if bad.any() else 0)


@pytest.mark.parametrize("small", [1e-12, 2.0 ** -100, 1e-38])
def test_long_sums_in_front_of_far_smaller_values(gpu, small):
    """Many heavy keys, then pages whose values are far smaller: the sums so far stay what they are."""
    seqs, kv, dim, steps = 64, 8, 64, 7500
    # page 0: scores of 0; page 1: scores 3.9 higher in powers of two; page 2: small values.  A run that begins in page 0 holds weights of almost 2^10.
    k = torch.zeros(3, kv, 16, dim, dtype=torch.int8, device="cuda")
    k[1, :, :, 0] = 127
    v = torch.full_like(k, 127)
    k_scale, v_scale = torch.full((3, kv), 1 / 127, device="cuda"), torch.tensor([1.0, 1.0, small], device="cuda")[:, None].repeat(1, kv)
    cache = gpu.Kv8Cache(k, v, k_scale, v_scale)
    number = torch.arange(steps, dtype=torch.int32, device="cuda") % 2
    number[6000:] = 2
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = gpu.Kv8Rows(number[None].repeat(seqs, 1).contiguous(), i32([steps * 16 - 1] * seqs), torch.arange(seqs + 1, dtype=torch.int32, device="cuda"), 1)
    q = torch.zeros(seqs, kv, dim, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 2.6875                                                   # 3.877 log 2
    out = cache.attention(rows, q, scale=1.0).double().cpu().numpy()
    e = math.exp(2.6875)
    want = 127 * (3000 + 3000 * e + 1500 * small) / (4500 + 3000 * e)
    # the weights' rounding and the matrix unit's additions (2^-23 of the sum each, 26,000 in a run at most, cut off), then bf16
    assert np.abs(out - want).max() <= want * (2.0 ** -10 + 26000 * 2.0 ** -23 + 2.0 ** -8)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("exponent", [-60, -110, -130])
def test_values_next_to_the_smallest_numbers(gpu, dtype, exponent):
    s = Setup(gpu, [(20, 2), (130, 1), (4000, 3)], 2, 64, 16, seed=82)
    for _ in range(2):
        s.plain.v_scale *= np.float32(2.0) ** np.float32(exponent / 2)
    s.pools[3].copy_(torch.from_numpy(s.plain.v_scale))
    check_relative(s, 4, dtype, s.normal(4, dtype))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("small", [2.0 ** -50, 1e-39, 1e-44])
def test_a_page_of_values_next_to_nothing_in_runs(gpu, dtype, small):
    s = Setup(gpu, [(520, 7), (384, 1), (700, 64), (5, 1)], 4, 64, 16, seed=62)
    for i, p in ((0, 3), (1, 0), (2, 40)):
        s.plain.v_scale[s.table[i, p]] = small
    s.pools[3].copy_(torch.from_numpy(s.plain.v_scale))
    s.batch = s.rows_of(1)
    check_relative(s, 16, dtype, s.normal(16, dtype))


@pytest.mark.parametrize("many", [0, 60])
def test_sequences_that_share_no_rows_in_any_order(gpu, many):
    """row_start that goes back between sequences which share no rows: the one that goes back is named, the others are served by every call."""
    seqs = [(20, 8), (0, 0), (50, 12)] + [(5, 0)] * many
    s = Setup(gpu, seqs, 2, 64, 16, seed=91, tail=20)
    start = np.array([30, 38, 4, 16] + [16] * many, np.int32)           # rows 30 .. 37, a step back, rows 4 .. 15
    (k, k64), (v, v64), (q, q64) = s.normal(2, "float32"), s.normal(2, "float32"), s.normal(4, "float32")
    batch = s.rows_of(12, start=start)
    turned = torch.full_like(q, 7.0)
    turns = gpu.rope_turns(10000.0, 64)
    s.cache.append(batch, k, v, turns=cuda(turns.view("int64")), q=q, q_out=turned)
    for i, (a, b) in ((0, (30, 38)), (2, (4, 16))):
        s.plain.append(s.table[i:i + 1], s.ctx[i:i + 1], [a, b], k64, v64, turns)
    s.same_cache()
    inside = np.zeros(s.rows, bool)
    inside[30:38] = inside[4:16] = True
    assert (host(turned)[~inside] == 7.0).all() and (host(turned)[inside] != 7.0).any(axis=(1, 2)).all()
    assert s.status.item() == 2
    out = torch.full_like(k, 7.0)
    s.cache.read(batch, k_out=out)
    assert (host(out)[~inside] == 7.0).all()
    for i, (a, b), c in ((0, (30, 38), 20), (2, (4, 16), 50)):
        want = s.plain.values("k", s.table[i], c + b - a)[c:]
        assert (np.abs(host(out)[a:b] - want) <= np.abs(want) * 2.0 ** -23).all()
    att = s.cache.attention(batch, q, torch.full_like(q, 7.0))
    assert (host(att)[~inside] == 7.0).all()
    for i, (a, b) in ((0, (30, 38)), (2, (4, 16))):
        want, mass, big, keys = s.plain.attention(s.table[i:i + 1], s.ctx[i:i + 1], [a, b], q64)
        bound = plain.attention_bound(want, mass, big, keys, 64, "float32", True)
        assert (np.abs(host(att) - want)[a:b] <= bound[a:b]).all()
