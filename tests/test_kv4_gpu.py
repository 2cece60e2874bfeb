"""The 4-bit key/value cache on the GPU against its definition in 64 bits: append, read, attention, weights of keys, eviction; and a step of a decoder with all of them."""
import math

import numpy as np
import pytest
import torch

import plain_kv4 as plain

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def cuda(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


class Setup:
    """A cache with random contents, sequences of given (context, new rows), pages in random order."""

    def __init__(self, lc, seqs, kv, dim, page, seed=0, spare=3, lead=0, tail=0):
        rng = self.rng = np.random.default_rng(seed)
        self.lc, self.seqs, self.kv, self.dim, self.page = lc, seqs, kv, dim, page
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
        self.rows = int(self.start[-1]) + tail
        # any bytes: slots that no row has been written to may hold any
        self.any = lambda *shape: rng.integers(0, 256, shape).astype(np.uint8)
        k, v = self.any(pages, kv, page, dim // 2), self.any(pages, kv, page, dim // 2)
        kb, vb = self.any(pages, kv, page, dim // 16), self.any(pages, kv, page, dim // 16)
        scales = lambda: np.exp(rng.normal(-4.5, 0.3, kv)).astype(np.float32)  # noqa: E731
        # what sequences hold: scales of ordinary sizes
        for i, (c, n) in enumerate(seqs):
            for slot in range(c + n):
                for b in (kb, vb):
                    b[self.table[i, slot // page], :, slot % page] = rng.integers(40, 88, (kv, dim // 16))
        self.plain = plain.PlainCache(k, v, kb, vb, scales(), scales())
        p = self.plain
        self.pools = [cuda(a) for a in (p.k, p.v, p.k_block, p.v_block, p.k_scale, p.v_scale)]
        self.cache = lc.Kv4Cache(*self.pools)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.batch = self.rows_of(max([n for _, n in seqs] + [0]))

    def rows_of(self, max_rows, ctx=None, start=None, table=None):
        return self.lc.Kv8Rows(cuda(self.table if table is None else table), cuda(self.ctx if ctx is None else ctx), cuda(self.start if start is None else start), max_rows, self.status)

    def normal(self, heads, dtype, scale=1.0, strided=0, rows=None):
        """Rows of values that the type holds: a tensor, and the same in 64 bits; strided: as a part of wider rows"""
        rows = self.rows if rows is None else rows
        x = torch.from_numpy(self.rng.normal(0, scale, (rows, heads, self.dim)).astype(np.float32)).to(DT[dtype])
        t = x.cuda()
        if strided:
            wide = torch.zeros(rows, heads * self.dim + strided, dtype=t.dtype, device="cuda")
            wide[:, :heads * self.dim] = t.reshape(rows, -1)
            t = wide[:, :heads * self.dim].unflatten(1, (heads, self.dim))
        return t, x.double().numpy()

    def check_pools(self):
        for name, t in zip(("k", "v", "k_block", "v_block"), self.pools):
            got, want = t.cpu().numpy(), getattr(self.plain, name)
            assert (got == want).all(), f"{name}: {(got != want).sum()} of {got.size} bytes"

    def turns(self, rot, theta=10000.0):
        t = self.lc.rope_turns(theta, rot)
        return t, torch.from_numpy(t.view("int64")).cuda()


def rotation_bound(want, dtype):
    """2^-23 of f32 results before the rounding; 16-bit ones: four roundings to f32, of products of at most the largest of two."""
    if dtype == "float32":
        return np.abs(want) * 2.0 ** -22 + 2.0 ** -40
    return np.abs(want) * plain.EPS[dtype] + np.abs(want).max(initial=0.0) * 2.0 ** -21 + plain.TINY[dtype]


SHAPES = [  # (kv, heads, dim, page, sequences of (context, new rows))
    (4, 32, 64, 16, [(700, 1)]),
    (8, 32, 128, 16, [(0, 1), (15, 1), (16, 1), (333, 1), (64, 1)]),
    (2, 2, 16, 32, [(31, 3), (5, 0), (0, 33)]),
    (1, 8, 128, 64, [(100, 17), (0, 70)]),
    (3, 6, 96, 16, [(7, 40), (200, 5)]),
    (2, 4, 256, 128, [(130, 9), (0, 2)]),
    (1, 1, 48, 256, [(255, 2), (1, 300)]),
    (2, 16, 112, 16, [(40, 4), (41, 4), (500, 4)]),
]
IDS = [f"{h}over{kv}x{d}p{p}" for kv, h, d, p, _ in SHAPES]


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_append_and_read(gpu, shape, dtype):
    kv, heads, dim, page, seqs = shape
    s = Setup(gpu, seqs, kv, dim, page, seed=dim + page, lead=2, tail=1)
    (k, k64), (v, v64), (q, q64) = s.normal(kv, dtype), s.normal(kv, dtype, 0.3), s.normal(heads, dtype)
    turns, on_gpu = s.turns(dim)
    q_out = torch.full_like(q, 7.0)
    assert s.cache.append(s.batch, k, v, turns=on_gpu, q=q, q_out=q_out) is q_out
    s.plain.append(s.table, s.ctx, s.start, k64, v64, turns)
    s.check_pools()
    inside = slice(s.start[0], s.start[-1])
    for i, (c, n) in enumerate(seqs):
        r = slice(s.start[i], s.start[i + 1])
        want = plain.rotate(q64[r], turns, c + np.arange(n))
        assert (np.abs(host(q_out)[r] - want) <= rotation_bound(want, dtype)).all()
    assert (host(q_out)[:s.start[0]] == 7.0).all() and (host(q_out)[s.start[-1]:] == 7.0).all()
    k_out, v_out = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    s.cache.read(s.batch, k_out, v_out)
    for name, out in (("k", k_out), ("v", v_out)):
        for i, (c, n) in enumerate(seqs):
            want = s.plain.values(name, s.table[i], c + n)[c:]
            assert (np.abs(host(out)[s.start[i]:s.start[i + 1]] - want) <= np.abs(want) * (plain.EPS[dtype] + 2.0 ** -24) + plain.TINY[dtype]).all()
        assert (np.delete(host(out), np.arange(inside.start, inside.stop), 0) == 7.0).all()
    assert s.status.item() == 0
    # earlier rows of the sequences are read as well
    only = torch.empty(seqs[0][0] + seqs[0][1], kv, dim, device="cuda")
    s.cache.read(gpu.Kv8Rows(cuda(s.table[:1]), cuda(np.zeros(1, np.int32)), cuda(np.array([0, len(only)], np.int32)), len(only), s.status), v_out=only)
    want = s.plain.values("v", s.table[0], len(only))
    assert (np.abs(host(only) - want) <= np.abs(want) * 2.0 ** -23).all()


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rot,strided", [(0, 0), (128, 1), (64, 0), (32, 8), (16, 0), (34, 0), (126, 3), (2, 0)])
def test_append_rotates_parts_of_the_head_at_other_positions(gpu, dtype, layout, rot, strided):
    kv, heads, dim = 2, 6, 128
    s = Setup(gpu, [(30, 5), (0, 20), (100, 1), (64, 0)], kv, dim, 16, seed=rot)
    (k, k64), (v, v64), (q, q64) = s.normal(kv, dtype, strided=strided), s.normal(kv, dtype, strided=strided), s.normal(heads, dtype, strided=strided)
    turns, on_gpu = s.turns(rot)
    positions = np.array([1_000_003, 0, 2 ** 40 + 17, 5], np.int64)
    q_out = s.cache.append(s.batch, k, v, turns=on_gpu if rot else None, q=q, positions=cuda(positions), layout=layout, magnitude=1.25)
    s.plain.append(s.table, s.ctx, s.start, k64, v64, turns, positions, layout, 1.25)
    s.check_pools()
    for i, (c, n) in enumerate(s.seqs):
        r = slice(s.start[i], s.start[i + 1])
        want = plain.rotate(q64[r], turns, positions[i] + np.arange(n), layout, 1.25)
        assert (np.abs(host(q_out)[r] - want) <= rotation_bound(want, dtype)).all()
        assert (host(q_out)[r][..., rot:] == q64[r][..., rot:].astype(np.float32)).all()


def test_append_rounds_ties_to_even_and_keeps_odd_numbers_out(gpu):
    """Values on borders between integers and between scales, infinities, NaN, zeros, numbers that no scale reaches; unturned, so that all are exact."""
    rng = np.random.default_rng(5)
    rows, kv, dim = 64, 2, 64
    s = Setup(gpu, [(0, rows)], kv, dim, 16)
    for scale in (1.0, 2.0 ** -6, 0.013, 2.0 ** -60, 2.0 ** 60):
        g = np.float32(scale)
        x = np.zeros((rows, kv, dim))
        for r in range(rows):
            for h in range(kv):
                for b in range(dim // 16):
                    code = rng.integers(1, 126)
                    step = plain.E4M3[code] * float(g)
                    x[r, h, 16 * b:16 * b + 16] = (rng.integers(-15, 16, 16) / 2.0) * step                # halves: ties
                    x[r, h, 16 * b] = 7.0 * float(g) * (plain.E4M3[code] if b % 2 else 0.5 * (plain.E4M3[code] + plain.E4M3[code + 1]))  # its scale, or the border of two
        x = x.astype(np.float32)
        x[3, 0, 5], x[4, 0, 6], x[5, 1, 7], x[6, 0, :16] = np.inf, -np.inf, np.nan, np.nan
        x[7, 0, :16], x[8, 0, :16], x[9, 1, 16:32], x[10] = 0.0, np.inf, 1e38, 1e-38
        x[11, 0, :16], x[12, 1] = 2.0 ** -149, -3.4e38
        s.plain.v_scale[:] = g
        s.plain.k_scale[:] = g
        s.pools[4].fill_(float(g))
        s.pools[5].fill_(float(g))
        s.cache.append(s.batch, cuda(x), cuda(x[:, ::-1]))
        s.plain.append(s.table, s.ctx, s.start, x, x[:, ::-1], [])
        s.check_pools()


def test_append_of_huge_keys_turns_beyond_f32(gpu):
    x = np.full((4, 1, 32), 3.0e38, np.float32)
    s = Setup(gpu, [(0, 4)], 1, 32, 16)
    s.pools[4].fill_(2.0 ** 60)
    s.plain.k_scale[:] = 2.0 ** 60
    turns, on_gpu = s.turns(32)
    s.cache.append(s.batch, cuda(x), cuda(x), turns=on_gpu)
    s.plain.append(s.table, s.ctx, s.start, x, x, turns)
    s.check_pools()


ATTENTION = SHAPES + [
    (2, 8, 64, 32, [(0, 150), (1000, 130)]),
    (2, 8, 128, 16, [(0, 300), (77, 140), (500, 64)]),
    (1, 2, 128, 16, [(2000, 1), (3, 1)]),
    (1, 16, 80, 64, [(300, 90)]),
    (4, 4, 128, 16, [(i * 37 % 400, 1) for i in range(40)]),
]
AIDS = [f"{h}over{kv}x{d}p{p}n{sum(n for _, n in q)}" for kv, h, d, p, q in ATTENTION]


def check_attention(s, out, lse, q64, dtype, scale=None, window=0, rows=None):
    want, wlse, mass, big, keys, weights = s.plain.attention(s.table, s.ctx, s.start, q64, scale, window)
    rows = np.concatenate([np.arange(s.start[i], s.start[i + 1]) for i in range(len(s.seqs))] + [np.zeros(0, int)]).astype(int) if rows is None else rows
    bound = plain.attention_bound(want, mass, big, keys, s.dim, dtype, dtype == "float32")
    err = np.abs(host(out).astype(np.float64) - want)
    assert (err[rows] <= bound[rows]).all(), f"worst {np.nanmax(err[rows] / bound[rows]):.2f} of the bound"
    if lse is not None:
        lerr = np.abs(host(lse).astype(np.float64) - wlse)[rows]
        lbound = (plain.score_bound(big, s.dim) + 2.0 ** -20 + np.abs(wlse) * 2.0 ** -22)[rows]
        assert (lerr <= lbound).all(), f"lse: worst {np.nanmax(lerr / lbound):.2f} of the bound"
    return weights


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("shape", ATTENTION, ids=AIDS)
def test_attention(gpu, shape, dtype):
    kv, heads, dim, page, seqs = shape
    s = Setup(gpu, seqs, kv, dim, page, seed=heads + dim, lead=1, tail=2)
    q, q64 = s.normal(heads, dtype)
    out, lse = torch.full_like(q, 7.0), torch.full((s.rows, heads), 7.0, device="cuda")
    s.cache.attention(s.batch, q, out, lse=lse)
    check_attention(s, out, lse, q64, dtype)
    for t in (out, lse):
        assert (host(t)[:s.start[0]] == 7.0).all() and (host(t)[s.start[-1]:] == 7.0).all()
    assert s.status.item() == 0


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("window", [1, 5, 16, 100, 129, 2 ** 40])
@pytest.mark.parametrize("seqs", [[(90, 2), (0, 3), (300, 1)], [(70, 150), (0, 200)]], ids=["few", "many"])
def test_attention_windows_scales_and_strides(gpu, seqs, window, dtype):
    kv, heads, dim = 2, 4, 128
    s = Setup(gpu, seqs, kv, dim, 16, seed=window % 1000)
    q, q64 = s.normal(heads, dtype, strided=4)
    wide = torch.full((s.rows, heads * dim + 8), 7.0, dtype=DT[dtype], device="cuda")
    out = wide[:, 8:].unflatten(1, (heads, dim))
    lse = torch.zeros(s.rows, heads + 3, device="cuda")[:, :heads]
    s.cache.attention(s.batch, q, out, lse=lse, scale=0.3, window=window)
    check_attention(s, out, lse, q64, dtype, 0.3, min(window, 10 ** 6))
    assert (host(wide)[:, :8] == 7.0).all()


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("seqs", [[(300, 1), (40, 1)], [(200, 160)]], ids=["few", "many"])
@pytest.mark.parametrize("what", ["far", "tiny", "outlier", "zeros", "large"])
def test_attention_of_queries_of_any_size(gpu, seqs, what, dtype):
    """Scores far from 0 (softmax takes the best key), queries next to f32's smallest, rows with one element far above the others, rows of zeros."""
    kv, heads, dim = 1, 4, 128
    s = Setup(gpu, seqs, kv, dim, 16, seed=3)
    q, _ = s.normal(heads, dtype)
    if what == "far":
        q[:, 1] *= 300.0
    elif what == "tiny":
        q[:, 1:] *= {"float32": 1e-37, "float16": 1e-7, "bfloat16": 1e-38}[dtype]
    elif what == "outlier":
        q[:, :, 5] *= 2.0 ** 11
    elif what == "zeros":
        q[:, 2] = 0.0
    else:
        q *= {"float32": 1e20, "float16": 1e4, "bfloat16": 1e20}[dtype]
    out, lse = torch.empty_like(q), torch.empty(s.rows, heads, device="cuda")
    scale = 1e-20 if what == "large" and dtype != "float16" else None
    s.cache.attention(s.batch, q, out, lse=lse, scale=scale)
    check_attention(s, out, lse, q.double().cpu().numpy(), dtype, scale)


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("seqs", [[(70, 3), (20, 1)], [(20, 200), (300, 30)]], ids=["few", "many"])
def test_rows_that_are_not_finite_are_nan_alone(gpu, seqs, dtype):
    s = Setup(gpu, seqs, 2, 64, 16, seed=4)
    q, _ = s.normal(4, dtype)
    q[1, 2, 3], q[2, 0, 0] = math.inf, math.nan
    out, lse = torch.empty_like(q), torch.empty(s.rows, 4, device="cuda")
    s.cache.attention(s.batch, q, out, lse=lse)
    bad = np.zeros((s.rows, 4), bool)
    bad[1, 2] = bad[2, 0] = True
    assert np.isnan(host(out)[bad]).all() and np.isnan(host(lse)[bad]).all()
    q64 = q.double().cpu().numpy()
    q64[1, 2] = q64[2, 0] = 0.0
    want, wlse, mass, big, keys, _ = s.plain.attention(s.table, s.ctx, s.start, q64)
    bound = plain.attention_bound(want, mass, big, keys, s.dim, dtype, dtype == "float32")
    assert (np.abs(host(out) - want) <= bound)[~bad].all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("seqs", [[(70, 3), (20, 2)], [(20, 150), (300, 30)]], ids=["few", "many"])
def test_bad_pages_and_sequences(gpu, seqs, dtype):
    """A page outside the pool: NaN in the rows that see it and nowhere else; a sequence outside its table: all of its rows."""
    s = Setup(gpu, seqs + [(5, 2)], 2, 64, 16, seed=6)
    q, q64 = s.normal(4, dtype)
    k, k64 = s.normal(2, dtype)
    table = s.table.copy()
    bad_slot = seqs[0][0] + seqs[0][1] - 1           # on the first sequence's last page
    table[0, bad_slot // 16] = 10 ** 6
    batch = s.rows_of(max(n for _, n in seqs), table=table)
    ctx = s.ctx.copy()
    ctx[2] = table.shape[1] * 16 - 1
    out, lse = torch.zeros_like(q), torch.zeros(s.rows, 4, device="cuda")
    s.cache.attention(batch, q, out, lse=lse)
    assert s.status.item() == 1
    slot = seqs[0][0] + np.arange(seqs[0][1])
    sees = np.zeros(s.rows, bool)
    sees[:seqs[0][1]] = slot >= bad_slot // 16 * 16
    assert np.isnan(host(out)[sees]).all() and np.isnan(host(lse)[sees]).all()
    check_attention(s, out, lse, q64, dtype, rows=np.nonzero(~sees)[0])
    mass = torch.zeros(3, 2, s.table.shape[1] * 16, device="cuda")
    good = torch.zeros_like(mass)
    s.cache.weights(batch, q, lse, mass)
    lse[torch.from_numpy(sees).cuda()] = math.nan
    s.cache.weights(s.batch, q, lse, good)
    assert torch.isfinite(mass).all() and (mass[1:] == good[1:]).all()
    # appends and reads
    s.status.zero_()
    before = [t.clone() for t in s.pools]
    s.cache.append(batch, k, k)
    assert s.status.item() == 1
    s.plain.append(s.table, s.ctx, s.start, k64, k64, [])
    for t, name, old in zip(s.pools, ("k", "v", "k_block", "v_block"), before):
        want = getattr(s.plain, name).copy()
        want[s.table[0, bad_slot // 16]] = old.cpu().numpy()[s.table[0, bad_slot // 16]]
        assert (t.cpu().numpy() == want).all()
    k_out = torch.zeros_like(k)
    s.cache.read(batch, k_out)
    assert np.isnan(host(k_out)[sees]).all() and np.isfinite(host(k_out)[~sees]).all()
    s.status.zero_()
    left = s.rows_of(2, ctx=ctx)
    q_out = s.cache.append(left, k, k, q=q, q_out=torch.full_like(q, 7.0))
    assert s.status.item() == 3 and (host(q_out)[s.start[2]:] == 7.0).all() and (host(q_out)[:s.start[2]] != 7.0).any()
    s.status.zero_()
    out.zero_()
    s.cache.attention(left, q, out, lse=lse)
    assert s.status.item() == 3 and np.isnan(host(out)[s.start[2]:]).all() and np.isnan(host(lse)[s.start[2]:]).all() and np.isfinite(host(out)[:s.start[2]]).all()
    s.status.zero_()
    mass.zero_()
    s.cache.weights(left, q, lse, mass)
    assert s.status.item() == 3 and (mass[2] == 0).all()


def mass_bound(mass, weights, big, group, shape, lse_off):
    """A weight is off by a factor of its score's error and its own lse's rounding, 2^-20 for exponentials and sums; the running sum by 2^-23."""
    out = np.zeros(shape)
    for i, r, h, lo, p in weights:
        out[i, h // group, lo:lo + len(p)] += p * (1.5 * (big[r, h] + lse_off[r, h]) + 2.0 ** -19)
    return out + np.abs(mass) * 2.0 ** -22 + 2.0 ** -100


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("shape", ATTENTION, ids=AIDS)
def test_weights(gpu, shape, dtype, window):
    kv, heads, dim, page, seqs = shape
    s = Setup(gpu, seqs, kv, dim, page, seed=heads + dim, lead=1, tail=2)
    q, q64 = s.normal(heads, dtype)
    _, wlse, _, big, _, weights = s.plain.attention(s.table, s.ctx, s.start, q64, None, window)
    lse = cuda(wlse.astype(np.float32))
    before = s.rng.random((len(seqs), kv, s.table.shape[1] * page + 5)).astype(np.float32)
    mass = cuda(before)
    want = before.astype(np.float64)
    for i, r, h, lo, p in weights:
        want[i, h // (heads // kv), lo:lo + len(p)] += p
    assert s.cache.weights(s.batch, q, lse, mass, window=window) is mass
    bound = mass_bound(want, weights, plain.score_bound(big, dim), heads // kv, want.shape, np.abs(wlse) * 2.0 ** -23)
    err = np.abs(host(mass) - want)
    assert (err <= bound).all(), f"worst {(err / bound).max():.2f} of the bound"
    assert s.status.item() == 0
    # twice the same, and the same again in a fresh tensor
    again = cuda(before)
    s.cache.weights(s.batch, q, lse, again, window=window)
    assert (again == mass).all()


def test_weights_need_room_and_leave_rows_out(gpu):
    s = Setup(gpu, [(60, 2), (20, 3)], 2, 64, 16)
    q, _ = s.normal(4, "bfloat16")
    out, lse = torch.empty_like(q), torch.empty(s.rows, 4, device="cuda")
    s.cache.attention(s.batch, q, out, lse=lse)
    wide = torch.zeros(2, 2, 100, device="cuda")
    s.cache.weights(s.batch, q, lse, wide[..., :61])          # the first sequence has 62 slots
    assert s.status.item() == 1 and (wide[0] == 0).all() and abs(wide[1].sum().item() - 12) < 1e-3 and (wide[..., 61:] == 0).all()
    lse[3] = math.nan                                          # a row that gives nothing
    wide.zero_()
    s.cache.weights(s.batch, q, lse, wide)
    assert abs(wide[0].sum().item() - 8) < 1e-3 and abs(wide[1].sum().item() - 8) < 1e-3
    turned = torch.zeros(2, 2, 100, device="cuda").transpose(0, 1)
    s.cache.weights(s.batch, q, lse, turned)
    assert (turned == wide).all()


EVICT = [  # (kv, dim, page, [(context, new)], keep, limit, recent, first)
    (2, 64, 16, [(700, 1), (10, 1), (100, 0), (101, 0)], 100, 100, 20, 3),
    (3, 128, 32, [(5000, 4), (1300, 1), (1281, 0), (1280, 0)], 1024, 1280, 128, 4),
    (1, 16, 16, [(40, 0)], 1, 1, 0, 0),
    (1, 256, 64, [(90, 7)], 96, 96, 1, 0),
    (2, 96, 256, [(300, 0), (0, 0), (2500, 0)], 60, 80, 30, 30),
    (1, 128, 128, [(9000, 0)], 8999, 8999, 0, 1),
]


@pytest.mark.parametrize("ties", ["none", "many", "odd"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: f"{c[0]}x{c[1]}keep{c[4]}")
def test_evict(gpu, case, ties):
    kv, dim, page, seqs, keep, limit, recent, first = case
    s = Setup(gpu, seqs, kv, dim, page, seed=keep)
    n, cap = len(seqs), max(s.table.shape[1] * page, limit) + 3
    mass = s.rng.lognormal(0, 2, (n, kv, cap)).astype(np.float32)
    if ties == "many":
        mass = np.floor(np.minimum(mass, 3.0))
    elif ties == "odd":
        mass = np.where(s.rng.random(mass.shape) < 0.3, s.rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0, 1e-45], np.float32), mass.shape), mass)
    mass = mass.astype(np.float32)
    on_gpu = cuda(mass)
    kept, ctx = s.cache.evict(s.batch, on_gpu, keep, limit=limit, recent=recent, first=first)
    kept, got = kept.cpu().numpy(), on_gpu.cpu().numpy()
    old = {name: getattr(s.plain, name).copy() for name in ("k", "v", "k_block", "v_block")}
    for i, (c, new) in enumerate(seqs):
        length = c + new
        assert ctx[i].item() == (keep if length > limit else length)
        for h in range(kv):
            stays = plain.evict(mass[i, h], length, keep, limit, recent, first)
            assert (kept[i, h, :len(stays)] == stays).all() and (kept[i, h, len(stays):] == -1).all()
            want = mass[i, h].copy()
            if length > limit:
                want[:length] = 0.0
                want[:keep] = mass[i, h][stays]
            assert np.array_equal(got[i, h], want, equal_nan=True)
            for name in old:
                for j, slot in enumerate(stays):
                    getattr(s.plain, name)[s.table[i, j // page], h, j % page] = old[name][s.table[i, slot // page], h, slot % page]
    s.check_pools()
    assert s.status.item() == 0


@pytest.mark.parametrize("length,keep", [(450_000, 300_000), (449_999, 17), (100, 50)])
def test_evict_of_contexts_beyond_shared_memory(gpu, length, keep):
    """Tables of more slots than a cluster's shared memory has sums for."""
    page, pages = 16, 30_000
    rng = np.random.default_rng(keep)
    table = rng.permutation(pages).astype(np.int32)[None]
    pools = [rng.integers(0, 256, (pages, 1, page, n)).astype(np.uint8) for n in (8, 8, 1, 1)]
    on_gpu = [cuda(a) for a in pools]
    cache = gpu.Kv4Cache(*on_gpu, torch.ones(1, device="cuda"), torch.ones(1, device="cuda"))
    rows = gpu.Kv8Rows(cuda(table), cuda(np.array([length], np.int32)), cuda(np.zeros(2, np.int32)), 0)
    mass = rng.lognormal(0, 2, (1, 1, page * pages)).astype(np.float32)
    got = cuda(mass)
    kept, ctx = cache.evict(rows, got, keep, recent=5, first=3)
    order = np.lexsort((np.arange(3, length - 5), -mass[0, 0, 3:length - 5]))[:keep - 8] + 3
    stays = np.sort(np.concatenate((np.arange(3), order, np.arange(length - 5, length))))
    assert ctx.item() == keep and (kept[0, 0].cpu().numpy() == stays).all()
    want = mass[0, 0].copy()
    want[:length] = 0.0
    want[:keep] = mass[0, 0][stays]
    assert (got[0, 0].cpu().numpy() == want).all()
    at = lambda slots: table[0][slots // page]  # noqa: E731
    for t, old in zip(on_gpu, pools):
        new = old.copy()
        new[at(np.arange(keep)), 0, np.arange(keep) % page] = old[at(stays), 0, stays % page]
        assert (t.cpu().numpy() == new).all()


def test_evict_leaves_bad_sequences_alone(gpu):
    s = Setup(gpu, [(100, 0), (100, 0), (100, 0), (100, 0)], 2, 64, 16)
    table, ctx = s.table.copy(), s.ctx.copy()
    table[0, 2], ctx[2] = -5, 10 ** 6
    mass = torch.rand(4, 2, 112, device="cuda")
    before = mass.clone()
    kept, new = s.cache.evict(s.rows_of(1, ctx=ctx, table=table), mass, 50)
    assert s.status.item() == 3
    assert (kept[0] == -1).all() and (kept[2] == -1).all() and (kept[1] >= 0).all() and new.tolist() == [100, 50, 10 ** 6, 50]
    assert (mass[0] == before[0]).all() and (mass[2] == before[2]).all()
    for t, name in zip(s.pools, ("k", "v", "k_block", "v_block")):
        for i in (0, 2):
            pages = s.table[i]
            assert (t.cpu().numpy()[pages] == getattr(s.plain, name)[pages]).all()
    s.status.zero_()
    s.cache.evict(s.batch, before[..., :99], 50)  # sums for fewer slots than there are
    assert s.status.item() == 4


@pytest.mark.parametrize("dtype", sorted(DT))
def test_a_decoder_that_evicts(gpu, dtype):
    """Prompts in chunks, then tokens; weights of all rows; eviction after each step; positions go on counting: every step against the plain cache."""
    kv, heads, dim, page, keep, limit, recent, first = 2, 8, 64, 16, 48, 64, 8, 2
    steps = [[40, 90], [30, 0], [1, 1], [1, 1], [5, 1], [1, 20]]
    s = Setup(gpu, [(0, 96), (0, 160)], kv, dim, page, seed=11)
    s.ctx = np.zeros(2, np.int32)
    turns, on_gpu = s.turns(dim)
    positions = np.zeros(2, np.int64)
    cap = s.table.shape[1] * page
    mass, plain_mass = torch.zeros(2, kv, cap, device="cuda"), np.zeros((2, kv, cap))
    for step in steps:
        s.seqs = [(int(c), n) for c, n in zip(s.ctx, step)]
        s.start = np.concatenate([[0], np.cumsum(step)]).astype(np.int32)
        s.rows = int(s.start[-1])
        batch = s.rows_of(max(step))
        (k, k64), (v, v64), (q, q64) = s.normal(kv, dtype), s.normal(kv, dtype), s.normal(heads, dtype)
        qr = s.cache.append(batch, k, v, turns=on_gpu, q=q, positions=cuda(positions))
        s.plain.append(s.table, s.ctx, s.start, k64, v64, turns, positions)
        s.check_pools()
        lse = torch.empty(s.rows, heads, device="cuda")
        out = s.cache.attention(batch, qr, lse=lse)
        q64 = qr.double().cpu().numpy()
        weights = check_attention(s, out, lse, q64, dtype)
        s.cache.weights(batch, qr, lse, mass)
        for i, r, h, lo, p in weights:
            plain_mass[i, h // (heads // kv), lo:lo + len(p)] += p
        got = host(mass)
        assert (np.abs(got - plain_mass) <= 1e-4 * plain_mass + 1e-5).all()   # scores of size 10, off by 1e-5: far inside
        kept, ctx = s.cache.evict(batch, mass, keep, limit=limit, recent=recent, first=first)
        old = {name: getattr(s.plain, name).copy() for name in ("k", "v", "k_block", "v_block")}
        for i, (c, n) in enumerate(s.seqs):
            for h in range(kv):
                stays = plain.evict(got[i, h], c + n, keep, limit, recent, first)
                assert (kept[i, h, :len(stays)].cpu().numpy() == stays).all()
                row = plain_mass[i, h].copy()
                plain_mass[i, h, :c + n] = 0.0
                plain_mass[i, h, :len(stays)] = row[stays]
                for name in old:
                    for j, slot in enumerate(stays):
                        getattr(s.plain, name)[s.table[i, j // page], h, j % page] = old[name][s.table[i, slot // page], h, slot % page]
        s.check_pools()
        positions += step
        s.ctx = ctx.cpu().numpy()
    assert s.status.item() == 0 and (s.ctx <= limit).all() and (positions == [78, 113]).all()


def test_captured_steps_follow_their_arrays(gpu):
    """One graph of append, attention, weights and eviction, replayed with other contexts, tables and rows."""
    kv, heads, dim, page = 2, 4, 64, 16
    s = Setup(gpu, [(20, 1), (50, 1), (33, 1)], kv, dim, page, seed=2)
    turns, on_gpu = s.turns(dim)
    q, k, v = (torch.zeros(3, h, dim, device="cuda") for h in (heads, kv, kv))
    positions = cuda(np.zeros(3, np.int64))
    lse, mass = torch.zeros(3, heads, device="cuda"), torch.zeros(3, kv, 80, device="cuda")
    qr, out = torch.zeros_like(q), torch.zeros_like(q)
    kept, ctx_out = torch.zeros(3, kv, 40, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    batch = s.batch
    table, ctx, start, _ = batch._kept
    ws = torch.empty(s.cache.attention_workspace(batch, q), dtype=torch.uint8, device="cuda")

    def step():
        s.cache.append(batch, k, v, turns=on_gpu, q=q, q_out=qr, positions=positions)
        s.cache.attention(batch, qr, out, lse=lse, workspace=ws)
        s.cache.weights(batch, qr, lse, mass)
        s.cache.evict(batch, mass, 30, limit=40, recent=4, kept=kept, ctx_out=ctx_out)
        ctx.copy_(ctx_out)
        positions.add_(1)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    torch.cuda.synchronize()
    assert (mass == 0).all() and s.status.item() == 0      # nothing ran
    ctx.copy_(cuda(s.ctx))
    for _ in range(3):
        fresh = [s.normal(h, "float32", rows=3) for h in (heads, kv, kv)]
        for t, (x, _) in zip((q, k, v), fresh):
            t.copy_(x)
        s.ctx, pos = ctx.cpu().numpy(), positions.cpu().numpy()
        s.seqs = [(int(c), 1) for c in s.ctx]
        before = host(mass).copy()
        graph.replay()
        torch.cuda.synchronize()
        s.plain.append(s.table, s.ctx, s.start, fresh[1][1], fresh[2][1], turns, pos)
        weights = check_attention(s, out, lse, qr.double().cpu().numpy(), "float32")
        for i, r, h, lo, p in weights:
            before[i, h // 2, lo:lo + len(p)] += p
        old = {name: getattr(s.plain, name).copy() for name in ("k", "v", "k_block", "v_block")}
        for i, (c, n) in enumerate(s.seqs):
            for h in range(kv):
                stays = kept[i, h].cpu().numpy()
                stays = stays[stays >= 0]
                assert len(stays) == (30 if c + n > 40 else c + n) and (np.diff(stays) > 0).all()
                assert np.abs(host(mass)[i, h, :len(stays)] - before[i, h][stays]).max() < 1e-4
                for name in old:
                    for j, slot in enumerate(stays):
                        getattr(s.plain, name)[s.table[i, j // page], h, j % page] = old[name][s.table[i, slot // page], h, slot % page]
        s.check_pools()
        assert (ctx.cpu().numpy() == [30 if c + 1 > 40 else c + 1 for c in s.ctx]).all()
    assert s.status.item() == 0


def test_two_streams_with_a_workspace_each(gpu):
    s = Setup(gpu, [(900, 1), (40, 1), (3000, 1)], 2, 128, 16, seed=9)
    q, _ = s.normal(8, "bfloat16")
    first = s.cache.attention(s.batch, q)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        outs = [s.cache.attention(s.batch, q, stream=st) for st in streams]
        torch.cuda.synchronize()
        assert all((o == first).all() for o in outs)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_far_pages_and_workspaces_of_larger_calls(gpu, dtype):
    """Pages whose bytes lie beyond 2^31, and a workspace that was asked for with a large call."""
    kv, dim, page, heads = 2, 128, 16, 4
    pages = 1_150_000                                                   # x 2048 bytes of keys
    pools = [torch.zeros(pages, kv, page, n, dtype=torch.uint8, device="cuda") for n in (dim // 2, dim // 2, dim // 16, dim // 16)]
    scales = torch.full((kv,), 0.02, device="cuda")
    cache = gpu.Kv4Cache(*pools, scales, scales)
    seqs = [(40, 3), (500, 1), (10, 200)]
    s = Setup(gpu, seqs, kv, dim, page, seed=8)
    far = (pages - 1 - np.arange(s.plain.k.shape[0])).astype(np.int32)
    for t, name in zip(pools, ("k", "v", "k_block", "v_block")):
        t[cuda(far.astype(np.int64))] = cuda(getattr(s.plain, name))
    s.plain.k_scale[:] = s.plain.v_scale[:] = np.float32(0.02)
    q, q64 = s.normal(heads, dtype)
    table = np.where(s.table >= 0, far[np.maximum(s.table, 0)], -1).astype(np.int32)
    ws = torch.empty(cache.attention_workspace(s.rows_of(200, table=table), q), dtype=torch.uint8, device="cuda")
    for max_rows in (200, 1):
        out, lse = torch.empty_like(q), torch.empty(s.rows, heads, device="cuda")
        cache.attention(s.rows_of(max_rows, table=table), q, out, lse=lse, workspace=ws)
        check_attention(s, out, lse, q64, dtype)
    k, k64 = s.normal(kv, dtype)
    cache.append(s.rows_of(200, table=table), k, k)
    s.plain.append(s.table, s.ctx, s.start, k64, k64, [])
    back = torch.empty_like(k)
    cache.read(s.rows_of(200, table=table), back)
    for i, (c, n) in enumerate(seqs):
        want = s.plain.values("k", s.table[i], c + n)[c:]
        assert (np.abs(host(back)[s.start[i]:s.start[i + 1]] - want) <= np.abs(want) * (plain.EPS[dtype] + 2.0 ** -24)).all()


def test_shared_pages_are_read_by_all(gpu):
    """Two sequences with the same first pages: attention and sums of each by itself."""
    s = Setup(gpu, [(64, 1), (64, 1)], 2, 64, 16, seed=12)
    s.table[1, :4] = s.table[0, :4]
    s.batch = s.rows_of(1)
    q, q64 = s.normal(4, "float32")
    out, lse = torch.empty_like(q), torch.empty(2, 4, device="cuda")
    s.cache.attention(s.batch, q, out, lse=lse)
    weights = check_attention(s, out, lse, q64, "float32")
    mass = torch.zeros(2, 2, 80, device="cuda")
    s.cache.weights(s.batch, q, lse, mass)
    want = np.zeros((2, 2, 80))
    for i, r, h, lo, p in weights:
        want[i, h // 2, lo:lo + len(p)] += p
    assert np.abs(host(mass) - want).max() < 1e-4
