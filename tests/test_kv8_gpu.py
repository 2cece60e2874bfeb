"""The 8-bit key/value cache on the GPU against its definition in 64 bits: append, read, attention; and a step of a decoder with all of them."""
import math

import numpy as np
import pytest
import torch

import plain_kv8 as plain

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def cuda(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


class Setup:
    """A cache with random contents, sequences of given (context, new rows), pages in random order."""

    def __init__(self, lc, seqs, kv, dim, page, seed=0, spare=3, lead=0, tail=0, status=True):
        rng = self.rng = np.random.default_rng(seed)
        self.seqs, self.kv, self.dim, self.page = seqs, kv, dim, page
        need = [-(-(c + n) // page) for c, n in seqs]
        width, pages = max(need + [1]), sum(need) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(seqs), width), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.ctx = np.array([c for c, _ in seqs], np.int32)
        self.start = (lead + np.concatenate([[0], np.cumsum([n for _, n in seqs])])).astype(np.int32)
        self.rows, self.tail = int(self.start[-1]) + tail, tail
        ints = lambda: rng.integers(-127, 128, (pages, kv, page, dim)).astype(np.int8)  # noqa: E731
        scales = lambda: np.exp(rng.normal(-4.5, 0.3, (pages, kv))).astype(np.float32)  # noqa: E731
        self.plain = plain.PlainCache(ints(), ints(), scales(), scales())
        self.pools = [cuda(a) for a in (self.plain.k, self.plain.v, self.plain.k_scale, self.plain.v_scale)]
        self.cache = lc.Kv8Cache(*self.pools)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.lc = lc
        self.batch = self.rows_of(max([n for _, n in seqs] + [0]))

    def rows_of(self, max_rows, ctx=None, start=None, table=None):
        return self.lc.Kv8Rows(cuda(self.table if table is None else table), cuda(self.ctx if ctx is None else ctx), cuda(self.start if start is None else start), max_rows, self.status)

    def normal(self, heads, dtype, scale=1.0, strided=0):
        """Rows of values that the type holds: a tensor, and the same in 64 bits; strided: as a part of wider rows"""
        x = torch.from_numpy(self.rng.normal(0, scale, (self.rows, heads, self.dim)).astype(np.float32)).to(DT[dtype])
        t = x.cuda()
        if strided:
            wide = torch.zeros(self.rows, heads * self.dim + strided, dtype=t.dtype, device="cuda")
            wide[:, :heads * self.dim] = t.reshape(self.rows, -1)
            t = wide[:, :heads * self.dim].unflatten(1, (heads, self.dim))
        return t, x.double().numpy()

    def inside(self):
        m = np.zeros(self.rows, bool)
        m[self.start[0]:self.start[-1]] = True
        return m

    def same_cache(self):
        for got, want, what in zip(self.pools, (self.plain.k, self.plain.v, self.plain.k_scale, self.plain.v_scale), ("k", "v", "k scale", "v scale")):
            assert np.array_equal(host(got), want), what


SEQS = {
    "one": [(700, 1)],
    "first": [(0, 1)],
    "ragged": [(0, 40), (5, 1), (37, 0), (16, 16), (31, 2), (0, 0), (130, 77)],
    "page ends": [(15, 1), (16, 1), (14, 3), (0, 16), (0, 17), (255, 2)],
    "many": [((i * 37) % 200, i % 3) for i in range(70)],
}


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("seqs", list(SEQS))
@pytest.mark.parametrize("kv,dim,page", [(4, 64, 16), (2, 128, 32), (3, 80, 128), (1, 256, 256)])
def test_append_and_read(gpu, dtype, seqs, kv, dim, page):
    s = Setup(gpu, SEQS[seqs], kv, dim, page, seed=len(seqs) + dim)
    heads = 2 * kv
    turns = gpu.rope_turns(10000.0, dim)
    (k, k64), (v, v64), (q, q64) = s.normal(kv, dtype), s.normal(kv, dtype, 0.3, strided=24), s.normal(heads, dtype, strided=1)
    out = s.cache.append(s.batch, k, v, turns=cuda(turns.view("int64")), q=q)
    s.plain.append(s.table, s.ctx, s.start, k64, v64, turns)
    s.same_cache()
    pos = np.concatenate([c + np.arange(n) for c, n in s.seqs]) if s.rows else np.zeros(0, int)
    want = plain.rotate(q64, turns, pos)
    # one rounding from 64 bits by way of f32
    err = np.abs(host(out) - want)
    assert (err <= np.abs(want) * (plain.EPS[dtype] / 2 + 2.0 ** -24) + plain.TINY[dtype] + 1e-14).all()
    assert s.status.item() == 0
    # everything that the sequences hold now, read back
    back = [(0, c + n) for c, n in s.seqs]
    start = np.concatenate([[0], np.cumsum([n for _, n in back])]).astype(np.int32)
    rows = s.rows_of(max(n for _, n in back), ctx=np.zeros(len(back), np.int32), start=start)
    ko, vo = (torch.zeros(int(start[-1]), kv, dim, dtype=DT[dtype], device="cuda") for _ in range(2))
    s.cache.read(rows, ko, vo)
    for got, which in ((ko, "k"), (vo, "v")):
        want = np.concatenate([s.plain.values(which, s.table[i], n) for i, (_, n) in enumerate(back)])
        assert (np.abs(host(got) - want) <= np.abs(want) * (plain.EPS[dtype] / 2 + 2.0 ** -24) + plain.TINY[dtype]).all()
    only = torch.zeros_like(ko)
    s.cache.read(rows, k_out=only)
    assert torch.equal(only, ko)


@pytest.mark.parametrize("rot", [0, 2, 32, 64])
def test_append_turns_a_part_of_the_dims(gpu, rot):
    s = Setup(gpu, [(3, 5), (20, 1)], 2, 64, 16)
    turns = gpu.rope_turns(500000.0, rot)
    (k, k64), (v, v64) = s.normal(2, "float32"), s.normal(2, "float32")
    s.cache.append(s.batch, k, v, turns=cuda(turns.view("int64")) if rot else None)
    s.plain.append(s.table, s.ctx, s.start, k64, v64, turns)
    s.same_cache()


def test_append_far_positions(gpu):
    s = Setup(gpu, [(1_000_003, 2), (262_143, 1)], 1, 64, 256)
    turns = gpu.rope_turns(10000.0, 64)
    (k, k64), (v, v64), (q, q64) = s.normal(1, "float32"), s.normal(1, "float32"), s.normal(2, "float32")
    out = s.cache.append(s.batch, k, v, turns=cuda(turns.view("int64")), q=q, q_out=q)  # in place
    assert out is q
    s.plain.append(s.table, s.ctx, s.start, k64, v64, turns)
    s.same_cache()
    want = plain.rotate(q64, turns, [1_000_003, 1_000_004, 262_143])
    assert (np.abs(host(out) - want) <= np.abs(want) * 2.0 ** -23 + 1e-14).all()


def test_scales_grow_token_by_token(gpu):
    """One token at a time into two pages, each larger than the last: earlier integers are rounded again at every step."""
    s = Setup(gpu, [(0, 1)], 2, 64, 16)
    s.table = np.array([[1, 0]], np.int32)
    for t in range(20):
        s.ctx = np.array([t], np.int32)
        (k, k64), (v, v64) = s.normal(2, "float32", 1.1 ** t), s.normal(2, "float32", 0.9 ** t)
        s.cache.append(s.rows_of(1), k, v)
        s.plain.append(s.table, s.ctx, s.start, k64, v64, [])
        s.same_cache()


def test_append_of_zeros_infinities_and_nan(gpu):
    s = Setup(gpu, [(4, 3), (0, 2), (16, 1)], 2, 64, 16)
    (k, k64), (v, v64) = s.normal(2, "float32"), s.normal(2, "float32")
    for x, x64 in ((k, k64), (v, v64)):
        for at, y in (((0, 0, 3), math.inf), ((1, 1, 5), -math.inf), ((2, 0, 7), math.nan)):
            x[at], x64[at] = y, y
        x[3:5], x64[3:5] = 0.0, 0.0                    # a new page of zeros: scale 0
        x[5, 0], x64[5, 0] = math.inf, math.inf        # nothing finite
    s.cache.append(s.batch, k, v)
    s.plain.append(s.table, s.ctx, s.start, k64, v64, [])
    s.same_cache()
    assert (host(s.pools[2])[s.table[1, 0]] == 0).all()


@pytest.mark.parametrize("size", [1e-30, 1e-37, 3e-41, 2e-44])
def test_append_next_to_the_smallest_numbers(gpu, size):
    """Magnitudes where a relative error of f32 is not one: the integers and scales are still those of the definition."""
    s = Setup(gpu, [(4, 30), (0, 2)], 2, 64, 16, seed=9)
    turns = gpu.rope_turns(10000.0, 64)
    (k, k64), (v, v64) = s.normal(2, "float32", size), s.normal(2, "float32", size)
    s.cache.append(s.batch, k, v, turns=cuda(turns.view("int64")))
    s.plain.append(s.table, s.ctx, s.start, k64, v64, turns)
    s.same_cache()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [3, 40])
def test_rows_given_to_several_sequences(gpu, dtype, new):
    """A row_start that goes back and forth: the sequence that shares no rows has its results, and nothing else is written."""
    s = Setup(gpu, [(20, new), (50, new), (9, new)], 2, 64, 16, tail=2)
    start = np.array([0, new, 0, 0], np.int32)      # the second goes back, the third has no rows: all rows are the first's
    q, q64 = s.normal(4, dtype)
    out = torch.full_like(q, 7.0)
    s.cache.attention(s.rows_of(new, start=start), q, out)
    want, mass, big, keys = s.plain.attention(s.table, s.ctx[:1], start[:2], q64)
    bound = plain.attention_bound(want, mass, big, keys, 64, dtype, dtype == "float32")
    assert (np.abs(host(out).astype(np.float64) - want)[:new] <= bound[:new]).all() and (host(out)[new:] == 7.0).all()
    assert s.status.item() == 2
    start = np.array([0, new, 2 * new, 0], np.int32)    # the last goes back: left alone
    s.status.zero_()
    s.cache.attention(s.rows_of(new, start=start), q, out.fill_(7.0))
    assert (host(out)[:2 * new] != 7.0).all() and (host(out)[2 * new:] == 7.0).all() and s.status.item() == 3


def test_results_made_for_another_stream(gpu):
    """Outputs and workspaces that a call makes for another stream are that stream's memory; a number for a stream makes none."""
    s = Setup(gpu, [(30, 2)], 2, 64, 16)
    (k, k64), (v, v64), (q, q64) = s.normal(2, "bfloat16"), s.normal(2, "bfloat16"), s.normal(4, "bfloat16")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    same = s.cache.append(s.batch, k, v, q=q, stream=side)
    out = s.cache.attention(s.batch, q, stream=side)
    side.synchronize()
    assert torch.equal(same, q) and torch.equal(out, s.cache.attention(s.batch, q))
    for call in (lambda: s.cache.append(s.batch, k, v, q=q, stream=side.cuda_stream), lambda: s.cache.attention(s.batch, q, torch.empty_like(q), stream=side.cuda_stream),
                 lambda: s.cache.attention(s.batch, q, workspace=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"), stream=side.cuda_stream)):
        with pytest.raises(ValueError):
            call()


def test_rows_outside_the_sequences_are_left_alone(gpu):
    s = Setup(gpu, [(3, 2), (18, 1)], 2, 64, 16, lead=2, tail=3)
    turns = gpu.rope_turns(10000.0, 64)
    (k, k64), (v, v64), (q, q64) = s.normal(2, "bfloat16"), s.normal(2, "bfloat16"), s.normal(4, "bfloat16")
    out = torch.full_like(q, 7.0)
    s.cache.append(s.batch, k, v, turns=cuda(turns.view("int64")), q=q, q_out=out)
    s.plain.append(s.table, s.ctx, s.start, k64, v64, turns)
    s.same_cache()
    assert (host(out)[~s.inside()] == 7.0).all() and (host(out)[s.inside()] != 7.0).any()
    ko = torch.full_like(k, 7.0)
    s.cache.read(s.batch, k_out=ko)
    assert (host(ko)[~s.inside()] == 7.0).all()
    o = torch.full_like(q, 7.0)
    s.cache.attention(s.batch, q, o)
    assert (host(o)[~s.inside()] == 7.0).all() and (host(o)[s.inside()] != 7.0).all()


def check_attention(s, heads, dtype, window=0, scale=None, q_scale=1.0, strided=0, max_rows=None, q=None):
    q, q64 = q or s.normal(heads, dtype, q_scale, strided)
    out = torch.full_like(q, math.nan)
    batch = s.batch if max_rows is None else s.rows_of(max_rows)
    s.cache.attention(batch, q, out, scale=scale, window=window)
    want, mass, big, keys = s.plain.attention(s.table, s.ctx, s.start, q64, scale, window)
    # the library may take either form for 16-bit types: the wider bound covers both
    bound = plain.attention_bound(want, mass, big, keys, s.dim, dtype, dtype == "float32")
    m = s.inside()
    err = np.abs(host(out).astype(np.float64) - want)[m]
    assert np.isfinite(err).all()
    assert (err <= bound[m]).all(), f"{(err / np.maximum(bound[m], 1e-300)).max():.2f} of the bound"
    assert s.status.item() == 0
    return out


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("seqs", list(SEQS))
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 4, 64, 16), (8, 2, 128, 32), (6, 2, 80, 64), (4, 1, 256, 128), (24, 2, 128, 16), (5, 5, 16, 256), (7, 1, 96, 16)])
def test_attention(gpu, dtype, seqs, heads, kv, dim, page):
    check_attention(Setup(gpu, SEQS[seqs], kv, dim, page, seed=len(seqs) + heads), heads, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 100, 100000, 2 ** 31 - 1])
def test_attention_windows(gpu, dtype, window):
    check_attention(Setup(gpu, [(500, 3), (0, 90), (99, 1), (64, 0), (63, 2)], 2, 64, 16), 4, dtype, window=window)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,kv,dim", [(16, 2, 128), (8, 8, 64)])
def test_attention_long_contexts_are_split(gpu, dtype, heads, kv, dim):
    check_attention(Setup(gpu, [(9001, 2), (40, 1), (4097, 5)], kv, dim, 64, seed=2), heads, dtype, strided=3)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 4, 128, 16), (8, 2, 128, 32), (6, 2, 64, 16), (4, 1, 96, 64)])
def test_attention_of_prompts(gpu, dtype, heads, kv, dim, page):
    check_attention(Setup(gpu, [(0, 300), (77, 130), (513, 64), (200, 1), (9, 33)], kv, dim, page, seed=3), heads, dtype)


@pytest.mark.parametrize("max_rows", [0, 1, 3, 4000])
def test_attention_whatever_max_rows_says(gpu, max_rows):
    for dtype in ("float32", "float16"):
        check_attention(Setup(gpu, [(100, 1), (20, 50), (0, 5)], 2, 128, 16, seed=4), 8, dtype, max_rows=max_rows)


@pytest.mark.parametrize("q_scale", [1e-30, 1e-6, 300.0, 1e20])
def test_attention_queries_of_any_size(gpu, q_scale):
    """The scale brings the scores back to about 1: queries far outside f16's range lose nothing."""
    s = Setup(gpu, [(300, 1), (40, 9)], 2, 64, 16, seed=5)
    check_attention(s, 4, "float32", q_scale=q_scale, scale=0.125 / q_scale)
    check_attention(s, 4, "bfloat16", q_scale=q_scale, scale=0.125 / q_scale)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads,kv,dim,new", [(4, 4, 128, 1), (8, 1, 64, 3), (4, 1, 256, 2), (4, 2, 96, 70)])
def test_attention_queries_with_an_outlier(gpu, dtype, heads, kv, dim, new):
    """One element of the queries a thousand times the others, where the keys are zero: the others' part of the scores keeps its bits."""
    s = Setup(gpu, [(200, new), (31, new)], kv, dim, 16, seed=16)
    s.plain.k[..., 5] = 0
    s.pools[0].copy_(torch.from_numpy(s.plain.k))
    q, q64 = s.normal(heads, dtype)
    q[..., 5], q64[..., 5] = 1000.0, 1000.0
    check_attention(s, heads, dtype, q=(q, q64))


def test_attention_of_zero_queries_and_zero_pages(gpu):
    s = Setup(gpu, [(60, 3)], 2, 64, 16, seed=6)
    for pool, scale in ((s.plain.k, s.plain.k_scale), (s.plain.v, s.plain.v_scale)):
        scale[s.table[0, 1]] = 0.0                      # a page of zeros among others
    for t, a in zip(s.pools, (s.plain.k, s.plain.v, s.plain.k_scale, s.plain.v_scale)):
        t.copy_(torch.from_numpy(a))
    q, q64 = s.normal(4, "float32")
    q[1], q64[1] = 0.0, 0.0
    check_attention(s, 4, "float32", q=(q, q64))


def test_attention_values_of_very_different_pages(gpu):
    """Scales of pages that differ by 2^40: a page's values count by its weights alone."""
    for dtype in ("float32", "bfloat16"):
        s = Setup(gpu, [(200, 1), (150, 20)], 2, 128, 16, seed=7)
        s.plain.v_scale *= np.exp2(s.rng.integers(-20, 21, s.plain.v_scale.shape)).astype(np.float32)
        s.pools[3].copy_(torch.from_numpy(s.plain.v_scale))
        check_attention(s, 8, dtype)


def test_attention_nothing_behind_the_end_counts(gpu):
    """Slots behind a sequence's last row, and pages that no sequence has: NaN scales there change nothing, nor do other integers."""
    s = Setup(gpu, [(33, 1), (15, 2)], 2, 64, 16, seed=8)
    q = s.normal(4, "float32")
    a = check_attention(s, 4, "float32", q=q).clone()
    used = np.unique(s.table[s.table >= 0])
    for scale in s.pools[2:]:
        free = torch.ones(scale.shape[0], dtype=torch.bool)
        free[used] = False
        scale[free.cuda()] = math.nan
    for pool in s.pools[:2]:
        pool[int(s.table[0, 2]), :, 2:] = 127
        pool[int(s.table[1, 1]), :, 1:] = -128
    assert torch.equal(a, check_attention(s, 4, "float32", q=q))


def test_pages_shared_between_sequences_are_read_by_both(gpu):
    s = Setup(gpu, [(64, 1), (64, 1), (64, 40)], 2, 64, 16, seed=9)
    s.table[1, :4] = s.table[0, :4]
    s.table[2, :2] = s.table[0, :2]
    s.batch = s.rows_of(40)
    check_attention(s, 4, "float32")


def test_results_repeat(gpu):
    s = Setup(gpu, [(3000, 1), (900, 2), (10, 300)], 2, 128, 16, seed=10)
    q, _ = s.normal(8, "bfloat16")
    first = s.cache.attention(s.batch, q)
    for _ in range(3):
        assert torch.equal(first, s.cache.attention(s.batch, q))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [1, 40])
def test_bad_pages_and_rows_are_kept_out(gpu, dtype, new):
    """Pages outside the pool, positions outside the table, row_start that is not ascending: nothing is read or written there, the status names
    the highest such sequence, and the others come out as ever."""
    seqs = [(50, new), (40, new), (30, new), (20, new)]
    good = Setup(gpu, seqs, 2, 64, 16, seed=11)
    q, q64 = good.normal(4, dtype)
    (k, _), (v, _) = good.normal(2, dtype), good.normal(2, dtype)
    exact, mass, big, keys = good.plain.attention(good.table, good.ctx, good.start, q64)
    bound = plain.attention_bound(exact, mass, big, keys, 64, dtype, dtype == "float32")
    n = lambda i: slice(int(good.start[i]), int(good.start[i + 1]))  # noqa: E731

    def as_ever(out, i):  # within the bound of any call: where contexts are cut, and with it the order of sums, goes by all sequences of a call
        return (np.abs(out[n(i)].astype(np.float64) - exact[n(i)]) <= bound[n(i)]).all()

    def attempt(table=None, ctx=None, start=None):
        s = Setup(gpu, seqs, 2, 64, 16, seed=11)
        b = s.rows_of(new, table=table, ctx=ctx, start=start)
        out, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
        s.cache.attention(b, q, out)
        a = s.status.item()
        s.status.zero_()
        s.cache.read(b, k_out=ko)
        r = s.status.item()
        s.status.zero_()
        before = [p.clone() for p in s.pools]
        s.cache.append(b, k, v)
        return host(out), host(ko), (a, r, s.status.item()), before, s.pools

    for page in (-1, -2 ** 31, good.plain.k.shape[0], 2 ** 31 - 1):
        table = good.table.copy()
        table[1, (40 + new - 1) // 16] = page           # the last row's page
        out, ko, status, before, after = attempt(table=table)
        assert status == (2, 2, 2)
        assert np.isnan(out[n(1)][-1]).all() and np.isnan(ko[n(1)][-1]).all()
        for i in (0, 2, 3):
            assert as_ever(out, i)
    for bad in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        ctx = good.ctx.copy()
        ctx[2] = bad
        out, ko, status, before, after = attempt(ctx=ctx)
        assert status == (3, 3, 3)
        assert np.isnan(out[n(2)]).all() and np.isnan(ko[n(2)]).all()
        for i in (0, 1, 3):
            assert as_ever(out, i)
        for x, y in zip(before, after):                  # its pages stay as they were
            used = [int(p) for p in good.table[2] if p >= 0]
            assert torch.equal(x[used], y[used])
    for start in ([0, new, 2 * new, 3 * new, 2 ** 31 - 1], [-5, new, 2 * new, 3 * new, 4 * new], [0, new, 2 * new, 4 * new + 1, 4 * new]):
        out, ko, status, before, after = attempt(start=np.array(start, np.int32))
        assert min(status) > 0
        assert as_ever(out, 1)
    # without a status word
    b = gpu.Kv8Rows(cuda(table), cuda(ctx), cuda(good.start), new)
    good.cache.attention(b, q)
    torch.cuda.synchronize()


def test_first_calls_of_a_process_inside_a_capture(gpu):
    """No call needs a run outside the capture first."""
    import os
    import subprocess
    import sys
    code = """
import torch, leafcutterllm_b200 as lc
i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
k, v = (torch.zeros(8, 2, 16, 128, dtype=torch.int8, device="cuda") for _ in range(2))
cache = lc.Kv8Cache(k, v, torch.zeros(8, 2, device="cuda"), torch.zeros(8, 2, device="cuda"))
table = torch.arange(8, dtype=torch.int32, device="cuda").reshape(1, 8)
turns = torch.from_numpy(lc.rope_turns(10000.0, 128).view("int64")).cuda()
q, x = torch.randn(80, 4, 128, device="cuda").bfloat16(), torch.randn(80, 2, 128, device="cuda").bfloat16()
tokens = torch.zeros(80, dtype=torch.int64, device="cuda")
one, many = lc.Kv8Rows(table, i32(80), i32(0, 1), 1), lc.Kv8Rows(table, i32(0), i32(0, 80), 80)
ws = [torch.empty(cache.attention_workspace(r, y), dtype=torch.uint8, device="cuda") for r, y in ((many, q), (one, q[:1]))]
out, out1, ro, kx = torch.empty_like(q), torch.empty_like(q[:1]), torch.empty_like(q), torch.empty_like(x)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    cache.append(many, x, x, turns=turns, q=q, q_out=ro)
    cache.attention(many, ro, out, workspace=ws[0])
    cache.append(one, x[:1], x[:1], turns=turns)
    cache.attention(one, ro[:1], out1, workspace=ws[1])
    cache.read(many, kx)
    lp = lc.token_logprobs_dev(out.reshape(80, -1), tokens, top=2)
g.replay()
torch.cuda.synchronize()
first = [t.clone() for t in (out, out1, kx, *lp)]
cache.append(many, x, x, turns=turns, q=q, q_out=ro)
cache.attention(many, ro, out, workspace=ws[0])
cache.append(one, x[:1], x[:1], turns=turns)
cache.attention(one, ro[:1], out1, workspace=ws[1])
cache.read(many, kx)
lp = lc.token_logprobs_dev(out.reshape(80, -1), tokens, top=2)
torch.cuda.synchronize()
assert all(torch.equal(a, b) and bool(torch.isfinite(a.float()).all()) for a, b in zip(first, (out, out1, kx, *lp)))
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_streams_and_graphs(gpu):
    """Calls on a stream of their own, two at once with a workspace each, and a captured step that is replayed for later positions."""
    s = Setup(gpu, [(40, 1), (300, 1)], 2, 128, 16, seed=12, spare=8)
    turns = cuda(gpu.rope_turns(10000.0, 128).view("int64"))
    q, _ = s.normal(8, "bfloat16")
    other, _ = s.normal(8, "bfloat16")
    want, want2 = s.cache.attention(s.batch, q), s.cache.attention(s.batch, other)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(a):
            x = s.cache.attention(s.batch, q)
        y = s.cache.attention(s.batch, other, stream=b)
        torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(y, want2)
    # a step: append and attend, the positions in tensors that grow; the longer sequence grows into a page that nobody has
    free = sorted(set(range(s.plain.k.shape[0])) - set(s.table[s.table >= 0].tolist()))
    s.table = np.concatenate([s.table, [[-1], [free[0]]]], 1).astype(np.int32)
    ctx = cuda(s.ctx)
    rows = gpu.Kv8Rows(cuda(s.table), ctx, cuda(s.start), 1, s.status)
    (k, k64), (v, v64) = s.normal(2, "bfloat16"), s.normal(2, "bfloat16")
    ws = torch.empty(s.cache.attention_workspace(rows, q), dtype=torch.uint8, device="cuda")
    qr, out = torch.empty_like(q), torch.empty_like(q)
    keep = [p.clone() for p in s.pools]

    def step():
        s.cache.append(rows, k, v, turns=turns, q=q, q_out=qr)
        s.cache.attention(rows, qr, out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for p, o in zip(s.pools, keep):
        p.copy_(o)
    results = []
    for t in range(5):
        graph.replay()
        results.append((out.clone(), [p.clone() for p in s.pools]))
        ctx += 1
    for p, o in zip(s.pools, keep):
        p.copy_(o)
    ctx.copy_(cuda(s.ctx))
    for t in range(5):
        step()
        assert torch.equal(out, results[t][0]) and all(torch.equal(p, o) for p, o in zip(s.pools, results[t][1]))
        ctx += 1
    assert s.status.item() == 0


def test_the_librarys_own_stream(gpu):
    """stream = NULL, as the other `_dev` calls: the library's stream, lc_dev_sync waits."""
    import ctypes as C
    s = Setup(gpu, [(90, 2)], 2, 64, 16, seed=13)
    q, _ = s.normal(4, "float32")
    want = s.cache.attention(s.batch, q)
    out = torch.empty_like(q)
    ws = torch.empty(s.cache.attention_workspace(s.batch, q), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    lib = gpu.load()
    gpu._capi.check(lib.lc_attention_kv8_dev(C.addressof(s.cache.struct), C.addressof(s.batch.struct), 0, q.shape[0], q.data_ptr(), 256, 4, 0.0, 0, out.data_ptr(), 256,
                                             ws.data_ptr(), ws.numel(), None))
    gpu._capi.check(lib.lc_dev_sync())
    assert torch.equal(out, want)


def test_refusals_on_the_gpu(gpu):
    s = Setup(gpu, [(90, 2)], 2, 64, 16)
    q, _ = s.normal(4, "float32")
    small = torch.empty(16, dtype=torch.uint8, device="cuda")
    with pytest.raises(gpu.LeafcutterError):
        s.cache.attention(s.batch, q, workspace=small)
    with pytest.raises(ValueError):
        s.cache.attention(s.batch, q.cpu())
    with pytest.raises(ValueError):
        s.cache.append(s.batch, q[:, :2].cpu(), q[:, :2].cpu())
    on_host = gpu.Kv8Cache(*[p.cpu() for p in s.pools])
    with pytest.raises(gpu.LeafcutterError):               # the library looks where the pools are
        gpu._capi.check(gpu.load().lc_kv8_read_dev(on_host._ref, s.batch._ref, 0, 2, q.data_ptr(), 256, None, 0, None))


def test_past_32_bits(gpu):
    """A pool of more than 2^32 bytes of keys: a sequence at its end."""
    pages, kv, page, dim = 2 ** 32 // (8 * 256 * 128) + 3, 8, 256, 128
    k, v = (torch.empty(pages, kv, page, dim, dtype=torch.int8, device="cuda") for _ in range(2))
    scales = [torch.full((pages, kv), 0.01, device="cuda") for _ in range(2)]
    cache = gpu.Kv8Cache(k, v, *scales)
    small = Setup(gpu, [(300, 3)], kv, dim, page, seed=14, spare=0)
    last = np.array([[pages - 1, pages - 2]], np.int32)
    for big, few in zip((k, v, *scales), small.pools):
        big[pages - 1], big[pages - 2] = few[int(small.table[0, 0])], few[int(small.table[0, 1])]
    rows = small.rows_of(3, table=last)
    q, _ = small.normal(16, "bfloat16")
    (nk, _), (nv, _) = small.normal(kv, "bfloat16"), small.normal(kv, "bfloat16")
    turns = cuda(gpu.rope_turns(10000.0, dim).view("int64"))
    a = small.cache.append(small.batch, nk, nv, turns=turns, q=q)
    b = cache.append(rows, nk, nv, turns=turns, q=q)
    assert torch.equal(a, b) and torch.equal(k[pages - 2], small.pools[0][int(small.table[0, 1])])
    assert torch.equal(small.cache.attention(small.batch, a), cache.attention(rows, a))
    outs = [torch.empty_like(nk) for _ in range(2)]
    small.cache.read(small.batch, k_out=outs[0])
    cache.read(rows, k_out=outs[1])
    assert torch.equal(*outs)


def test_a_decoders_step(gpu):
    """A prompt, then tokens one by one, through append, attention, a head and log probabilities, against the same in 64 bits."""
    rng = np.random.default_rng(15)
    heads, kv, dim, page, vocab, hidden = 8, 2, 64, 16, 500, 96
    s = Setup(gpu, [(0, 45), (0, 7)], kv, dim, page, seed=15)
    s.table = np.arange(10, dtype=np.int32).reshape(2, 5)[:, ::-1].copy()
    pools = [torch.zeros(10, kv, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.zeros(10, kv, device="cuda") for _ in range(2)]
    s.pools, s.cache = pools, gpu.Kv8Cache(*pools)
    s.plain = plain.PlainCache(*[host(p) for p in pools])
    wq, wk, wv = (rng.normal(0, hidden ** -0.5, (hidden, n * dim)) for n in (heads, kv, kv))
    head = rng.normal(0, 2 * (heads * dim) ** -0.5, (heads * dim, vocab))
    emb = rng.normal(0, 1, (vocab, hidden))
    turns = gpu.rope_turns(10000.0, dim)
    ctx, new = np.zeros(2, np.int32), np.array([45, 7])
    tokens = rng.integers(0, vocab, 52)
    for step in range(6):
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        rows = gpu.Kv8Rows(cuda(s.table), cuda(ctx), cuda(start), int(new.max()), s.status)
        x = emb[tokens]
        q, k, v = ((x @ w).astype(np.float32).reshape(len(tokens), -1, dim) for w in (wq, wk, wv))
        qr = s.cache.append(rows, cuda(k), cuda(v), turns=cuda(turns.view("int64")), q=cuda(q))
        att = s.cache.attention(rows, qr)
        logits = (att.reshape(len(tokens), -1).double() @ cuda(head)).float()
        asked = rng.integers(0, vocab, len(tokens))
        lp, ent, tl, ti = gpu.token_logprobs_dev(logits, cuda(asked), top=4)
        s.plain.append(s.table, ctx, start, k.astype(np.float64), v.astype(np.float64), turns)
        s.same_cache()
        pos = np.concatenate([ctx[i] + np.arange(new[i]) for i in range(2)])
        want, mass, big, keys = s.plain.attention(s.table, ctx, start, plain.rotate(q.astype(np.float64), turns, pos))
        # the queries' own rounding to f32 moves a score by 2^-24 of `big`, which the bound's factor holds
        bound = plain.attention_bound(want, mass, big, keys, dim, "float32", True)
        err = np.abs(host(att) - want)
        assert (err <= bound).all()
        # a logit is off by at most the sum of |head| times the output's bound, and its rounding; log probabilities by twice the largest of them
        w_logits = want.reshape(len(tokens), -1) @ head
        off = (bound.reshape(len(tokens), -1) @ np.abs(head)).max(1) + np.abs(w_logits).max(1) * 2.0 ** -23
        w = plain.logprobs(w_logits, asked, 4)
        assert (np.abs(host(lp) - w[0]) <= 2 * off + 1e-5).all()
        assert (np.abs(host(tl) - w[2]) <= 2 * off[:, None] + 1e-5).all()
        # entropy moves by at most twice the logits' error times (its logs' spread)
        assert (np.abs(host(ent) - w[1]) <= 4 * off * (np.abs(w_logits).max(1) * 2 + 1) + 1e-5).all()
        ctx, new = ctx + new.astype(np.int32), np.array([1, 1])
        tokens = host(ti)[start[1:] - 1, 0]
    assert s.status.item() == 0
