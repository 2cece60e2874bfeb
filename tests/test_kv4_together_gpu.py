"""Calls over the 4-bit cache one after the other and at the same time, each one's results against the definition: eviction of as many sequences as there may be, a captured step's weights before and
after its eviction, streams with workspaces of their own, results that repeat, tables far wider than what sequences hold."""
import numpy as np
import pytest
import torch

import plain_kv4 as plain
from test_kv4_gpu import DT, Setup, check_attention, cuda, host, mass_bound

pytestmark = pytest.mark.gpu


def check_evict(s, before, mass, kept, ctx, keep, limit, recent, first):
    """Slots, sums and rows that stay, of sums as they were `before`; the plain cache follows."""
    old = {n: getattr(s.plain, n).copy() for n in ("k", "v", "k_block", "v_block")}
    want, want_kept, want_ctx = before.copy(), np.full((len(s.seqs), s.kv, limit), -1), []
    for i, (c, n) in enumerate(s.seqs):
        cut = c + n > limit
        want_ctx.append(keep if cut else c + n)
        for h in range(s.kv):
            stays = plain.evict(before[i, h], c + n, keep, limit, recent, first)
            want_kept[i, h, :len(stays)] = stays
            if not cut:
                continue
            to = np.arange(keep)
            want[i, h, :c + n] = 0.0
            want[i, h, :keep] = before[i, h, stays]
            for name, was in old.items():
                getattr(s.plain, name)[s.table[i][to // s.page], h, to % s.page] = was[s.table[i][stays // s.page], h, stays % s.page]
    assert (kept.cpu().numpy() == want_kept).all() and (ctx.cpu().numpy() == want_ctx).all() and (host(mass) == want).all()
    s.check_pools()


def check_mass(s, mass, weights, q64, wlse, big):
    """Sums of weights under the lse that attention on the GPU gave: a weight is off by its score's error, by the lse's (a score's error, 2^-20 and two roundings of lse to f32) and by lse's rounding in
    powers of two."""
    want, group = np.zeros(mass.shape), q64.shape[1] // s.kv
    for i, r, h, lo, p in weights:
        want[i, h // group, lo:lo + len(p)] += p
    bound = mass_bound(want, weights, 2 * plain.score_bound(big, s.dim) + 2.0 ** -20, group, want.shape, np.abs(wlse) * 2.0 ** -21)
    assert want.sum() > 0.9 * q64.shape[0] * q64.shape[1] and (np.abs(host(mass) - want) <= bound).all()


@pytest.mark.parametrize("kv", [1, 3])
def test_eviction_of_as_many_sequences_as_there_may_be(gpu, kv):
    rng = np.random.default_rng(kv)
    s = Setup(gpu, [(int(c), 0 if i % 5 == 3 else 1) for i, c in enumerate(rng.integers(0, 60, 4096))], kv, 32, 16, seed=kv)
    before = np.floor(rng.lognormal(0, 1, (4096, kv, 64)) * 4.0).astype(np.float32)      # with ties
    mass = cuda(before)
    kept, ctx = s.cache.evict(s.batch, mass, 20, limit=25, recent=2, first=1)
    check_evict(s, before, mass, kept, ctx, 20, 25, 2, 1)
    assert s.status.item() == 0


@pytest.mark.parametrize("dtype,dim", [("float32", 48), ("float16", 80), ("bfloat16", 144)])
@pytest.mark.parametrize("rows", [1, 70])
def test_a_captured_step_s_weights_and_what_its_eviction_makes_of_them(gpu, dtype, dim, rows):
    s = Setup(gpu, [(30, rows)], 2, dim, 16, seed=dim)
    q, q64 = s.normal(6, dtype)
    capacity = s.table.shape[1] * 16
    out, lse, mass = torch.empty_like(q), torch.empty(rows, 6, device="cuda"), torch.zeros(1, 2, capacity, device="cuda")
    seen = torch.empty_like(mass)
    kept, ctx = torch.empty(1, 2, 20, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(s.cache.attention_workspace(s.batch, q), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.cache.attention(s.batch, q, out, lse=lse, workspace=ws)
        s.cache.weights(s.batch, q, lse, mass)
        seen.copy_(mass)
        s.cache.evict(s.batch, mass, 20, recent=3, kept=kept, ctx_out=ctx)
    graph.replay()
    torch.cuda.synchronize()
    weights = check_attention(s, out, lse, q64, dtype)
    _, wlse, _, big, _, _ = s.plain.attention(s.table, s.ctx, s.start, q64)
    check_mass(s, seen, weights, q64, wlse, big)
    check_evict(s, host(seen), mass, kept, ctx, 20, 20, 3, 0)


@pytest.mark.parametrize("seqs", [[(900, 1), (40, 1), (3000, 1)], [(900, 90), (40, 64)]], ids=["few", "many"])
@pytest.mark.parametrize("dtype", sorted(DT))
def test_streams_with_workspaces_of_their_own(gpu, seqs, dtype):
    s = Setup(gpu, seqs, 2, 128, 16, seed=9)
    queries = [s.normal(8, dtype)[0] for _ in range(2)]
    first = [s.cache.attention(s.batch, q) for q in queries]
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [torch.empty(s.cache.attention_workspace(s.batch, queries[0]), dtype=torch.uint8, device="cuda") for _ in streams]
    outs = [torch.empty_like(q) for q in queries]
    torch.cuda.synchronize()
    for _ in range(20):
        for out in outs:
            out.fill_(7.0)
        torch.cuda.synchronize()
        for q, out, ws, st in zip(queries, outs, spaces, streams):
            s.cache.attention(s.batch, q, out, workspace=ws, stream=st)
        torch.cuda.synchronize()
        assert all((a == b).all() for a, b in zip(outs, first))


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("kv,heads,dim,seqs", [(2, 8, 128, [(900, 1), (40, 1), (3000, 4)]), (1, 8, 64, [(500, 150), (0, 40)]), (2, 4, 256, [(700, 9)])], ids=str)
def test_results_repeat(gpu, kv, heads, dim, seqs, dtype):
    s = Setup(gpu, seqs, kv, dim, 32, seed=11)
    q, _ = s.normal(heads, dtype)
    results = []
    for fill in (0.0, 7.0, 255.0):
        ws = torch.full((s.cache.attention_workspace(s.batch, q),), int(fill), dtype=torch.uint8, device="cuda")   # whatever a workspace holds
        lse, mass = torch.empty(s.rows, heads, device="cuda"), torch.ones(len(seqs), kv, s.table.shape[1] * 32, device="cuda")
        out = s.cache.attention(s.batch, q, lse=lse, workspace=ws)
        results.append((out, lse, s.cache.weights(s.batch, q, lse, mass)))
    assert all(torch.equal(a, b) for other in results[1:] for a, b in zip(results[0], other))


@pytest.mark.parametrize("width", [40, 5000, 20_000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tables_far_wider_than_what_sequences_hold(gpu, width, dtype):
    """Kernels and blocks are chosen by the tables; what stands behind a sequence's last page is not looked at."""
    s = Setup(gpu, [(300, 1), (10, 40), (0, 3), (500, 0)], 2, 64, 16, seed=13)
    table = np.full((4, width), 2 ** 31 - 1, np.int32)
    for i, (c, n) in enumerate(s.seqs):
        pages = -(-(c + n) // 16)
        table[i, :pages] = s.table[i, :pages]
    s.table = table
    s.batch = s.rows_of(40)
    q, q64 = s.normal(4, dtype)
    out, lse = torch.empty_like(q), torch.empty(s.rows, 4, device="cuda")
    s.cache.attention(s.batch, q, out, lse=lse)
    weights = check_attention(s, out, lse, q64, dtype)
    _, wlse, _, big, _, _ = s.plain.attention(s.table, s.ctx, s.start, q64)
    mass = torch.zeros(4, 2, 16 * width, device="cuda")
    s.cache.weights(s.batch, q, lse, mass)
    check_mass(s, mass, weights, q64, wlse, big)
    before = s.rng.lognormal(0, 2, mass.shape).astype(np.float32)
    mass = cuda(before)
    kept, ctx = s.cache.evict(s.batch, mass, 30, limit=45, recent=4, first=2)
    check_evict(s, before, mass, kept, ctx, 30, 45, 4, 2)
    assert s.status.item() == 0
