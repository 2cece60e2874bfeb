"""What the calls over the 4-bit key/value cache and of rotary positions refuse, and the scaled rotation tables: host code, no GPU.

Every refusal comes before the library looks for a device, so the pointers here are never read."""
import ctypes as C
import math

import numpy as np
import pytest

P = 1 << 20  # an address that is 16-byte aligned and never read
BF16, F32 = 30, 0


def cache(lc, **over):
    d = dict(k_dev=P, v_dev=P, k_block_dev=P, v_block_dev=P, k_scale_dev=P, v_scale_dev=P, n_pages=4, n_kv_heads=2, page_tokens=16, head_dim=64)
    d.update(over)
    return lc._capi.Kv4CacheStruct(**d)


def rows(lc, **over):
    d = dict(page_table_dev=P, ctx_dev=P, row_start_dev=P, status_dev=None, n_seqs=2, table_width=3, max_rows=1, reserved=0)
    d.update(over)
    return lc._capi.Kv8RowsStruct(**d)


def append(lc, c=None, r=None, typ=F32, n=2, pos=None, k=P, ks=128, v=P, vs=128, q=None, qs=0, qo=None, os=0, heads=0, turns=P, rot=64, layout=0, mag=1.0):
    return lc.load().lc_kv4_append_dev(C.byref(c or cache(lc)), C.byref(r or rows(lc)), typ, n, pos, k, ks, v, vs, q, qs, qo, os, heads, turns, rot, layout, mag, None)


def read(lc, c=None, r=None, typ=F32, n=2, k=P, ks=128, v=P, vs=128):
    return lc.load().lc_kv4_read_dev(C.byref(c or cache(lc)), C.byref(r or rows(lc)), typ, n, k, ks, v, vs, None)


def attend(lc, c=None, r=None, typ=F32, n=2, q=P, qs=256, heads=4, scale=0.0, window=0, out=P, os=256, lse=None, ls=4, ws=P, wb=1 << 40):
    return lc.load().lc_attention_kv4_dev(C.byref(c or cache(lc)), C.byref(r or rows(lc)), typ, n, q, qs, heads, scale, window, out, os, lse, ls, ws, wb, None)


def weigh(lc, c=None, r=None, typ=F32, n=2, q=P, qs=256, heads=4, scale=0.0, window=0, lse=P, ls=4, mass=P, ms=96, mh=48, cap=48):
    return lc.load().lc_kv4_weights_dev(C.byref(c or cache(lc)), C.byref(r or rows(lc)), typ, n, q, qs, heads, scale, window, lse, ls, mass, ms, mh, cap, None)


def evict(lc, c=None, r=None, mass=P, ms=96, mh=48, cap=48, keep=16, limit=32, recent=4, first=4, kept=P, ctx=P + 64):
    return lc.load().lc_kv4_evict_dev(C.byref(c or cache(lc)), C.byref(r or rows(lc)), mass, ms, mh, cap, keep, limit, recent, first, kept, ctx, None)


def rope(lc, typ=F32, n=2, pos=P, turns=P, rot=64, dim=64, layout=0, inverse=0, mag=1.0, x=P, xs=256, xo=P, xos=256, xh=4, y=None, ys=0, yo=None, yos=0, yh=0):
    return lc.load().lc_rope_dev(typ, n, pos, turns, rot, dim, layout, inverse, mag, x, xs, xo, xos, xh, y, ys, yo, yos, yh, None)


BAD_CACHE = [dict(k_dev=None), dict(v_dev=None), dict(k_block_dev=None), dict(v_block_dev=None), dict(k_scale_dev=None), dict(v_scale_dev=None), dict(k_dev=P + 8), dict(v_dev=P + 1),
             dict(k_block_dev=P + 4), dict(v_block_dev=P + 8), dict(n_pages=0), dict(n_kv_heads=0), dict(n_kv_heads=1025), dict(head_dim=0), dict(head_dim=72), dict(head_dim=272), dict(page_tokens=0),
             dict(page_tokens=8), dict(page_tokens=24), dict(page_tokens=512)]
BAD_ROWS = [dict(n_seqs=-1), dict(n_seqs=4097), dict(table_width=-1), dict(table_width=1 << 30), dict(max_rows=-1), dict(page_table_dev=None),
            dict(ctx_dev=None), dict(row_start_dev=None)]


@pytest.mark.parametrize("call", [append, read, attend, weigh, evict])
@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_caches_are_refused(lc, call, bad):
    assert call(lc, c=cache(lc, **bad)) == lc._capi.LC_ERR_INVALID
    assert lc.load().lc_last_error()


@pytest.mark.parametrize("call", [append, read, attend, weigh, evict])
@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_bad_rows_are_refused(lc, call, bad):
    assert call(lc, r=rows(lc, **bad)) == lc._capi.LC_ERR_INVALID


@pytest.mark.parametrize("call", [append, read, attend, weigh])
def test_types_and_row_counts(lc, call):
    assert call(lc, typ=8) == lc._capi.LC_ERR_UNSUPPORTED
    assert call(lc, n=-1) == lc._capi.LC_ERR_INVALID
    assert call(lc, n=(1 << 24) + 1) == lc._capi.LC_ERR_INVALID
    assert call(lc, n=0) == lc._capi.LC_OK                          # nothing to do, even without a device
    assert call(lc, r=rows(lc, n_seqs=0)) == lc._capi.LC_OK


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(ks=127), dict(vs=0), dict(rot=63), dict(rot=66), dict(rot=-2), dict(turns=None), dict(layout=2), dict(layout=-1),
                                 dict(mag=math.inf), dict(mag=math.nan), dict(q=P, qo=None, qs=256, os=256, heads=4), dict(q=P, qo=P, qs=255, os=256, heads=4),
                                 dict(q=P, qo=P, qs=256, os=255, heads=4), dict(q=P, qo=P, qs=256, os=256, heads=0), dict(q=P, qo=P, qs=256, os=300, heads=4)], ids=str)
def test_append_refuses(lc, bad):
    assert append(lc, **bad) == lc._capi.LC_ERR_INVALID


@pytest.mark.parametrize("bad", [dict(ks=127), dict(vs=127)], ids=str)
def test_read_refuses(lc, bad):
    assert read(lc, **bad) == lc._capi.LC_ERR_INVALID


ATTEND = [dict(q=None), dict(qs=255), dict(heads=0), dict(heads=3), dict(heads=65538), dict(window=-1), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan)]


@pytest.mark.parametrize("bad", ATTEND + [dict(out=None), dict(os=1), dict(lse=P, ls=3)], ids=str)
def test_attention_refuses(lc, bad):
    assert attend(lc, **bad) == lc._capi.LC_ERR_INVALID


@pytest.mark.parametrize("bad", ATTEND + [dict(lse=None), dict(ls=3), dict(mass=None), dict(cap=-1), dict(cap=49), dict(ms=47), dict(ms=48), dict(mh=0)], ids=str)
def test_weights_refuse(lc, bad):
    assert weigh(lc, **bad) == lc._capi.LC_ERR_INVALID


@pytest.mark.parametrize("bad", [dict(mass=None), dict(kept=None), dict(ctx=None), dict(ctx=P), dict(keep=0), dict(keep=-1), dict(keep=7), dict(keep=33), dict(limit=49), dict(recent=-1), dict(first=-1),
                                 dict(recent=2 ** 31 - 1, first=2 ** 31 - 1), dict(cap=49), dict(ms=48), dict(mh=47)], ids=str)
def test_eviction_refuses(lc, bad):
    assert evict(lc, **bad) == lc._capi.LC_ERR_INVALID


def test_eviction_of_nothing(lc):
    assert evict(lc, r=rows(lc, n_seqs=0)) == lc._capi.LC_OK


@pytest.mark.parametrize("bad", [dict(pos=None), dict(turns=None), dict(rot=63), dict(rot=66), dict(rot=-2), dict(dim=0), dict(dim=1025, rot=0), dict(layout=2), dict(mag=math.nan), dict(mag=1e31), dict(x=None),
                                 dict(xo=None), dict(xs=255), dict(xos=255), dict(xh=0), dict(xh=65537), dict(xos=260), dict(n=-1), dict(n=(1 << 24) + 1),
                                 dict(y=P, ys=256, yo=None, yos=256, yh=4), dict(y=P, ys=255, yo=P, yos=256, yh=4), dict(y=P, ys=256, yo=P, yos=256, yh=0)], ids=str)
def test_rope_refuses(lc, bad):
    assert rope(lc, **bad) == lc._capi.LC_ERR_INVALID


def test_rope_of_nothing_and_of_other_types(lc):
    assert rope(lc, n=0) == lc._capi.LC_OK
    assert rope(lc, typ=8) == lc._capi.LC_ERR_UNSUPPORTED


@pytest.mark.parametrize("bad", [dict(kind="linear", factor=0.5), dict(kind="linear", factor=math.inf), dict(kind="yarn", factor=4.0, original=0), dict(kind="yarn", factor=4.0, original=2048, fast=1.0, slow=2.0),
                                 dict(kind="llama3", factor=4.0, original=2048, fast=4.0, slow=-1.0), dict(kind="ntk", factor=4.0, rot=2), dict(rot=7), dict(rot=-2), dict(theta=0.5),
                                 dict(theta=math.nan), dict(kind="yarn", factor=2.0, original=2048, theta=1.0)], ids=str)
def test_scaled_tables_refuse(lc, bad):
    d = dict(kind="none", theta=10000.0, rot=64, factor=1.0, original=0, fast=0.0, slow=0.0)
    d.update(bad)
    with pytest.raises(lc.LeafcutterError):
        lc.rope_turns_scaled(d["theta"], d["rot"], d["kind"], d["factor"], d["original"], d["fast"], d["slow"])


def test_unknown_names_are_refused(lc):
    with pytest.raises(ValueError):
        lc.rope_turns_scaled(10000.0, 64, "other")
    with pytest.raises(ValueError):
        lc.device._layout("other")


@pytest.mark.parametrize("rot", [0, 2, 64, 96, 128])
@pytest.mark.parametrize("kind,factor,original", [("none", 1.0, 0), ("linear", 4.0, 0), ("ntk", 3.5, 0), ("yarn", 16.0, 8192), ("yarn", 2.0, 100), ("llama3", 8.0, 8192), ("llama3", 1.0, 2048)])
def test_scaled_tables(lc, kind, factor, original, rot):
    """Frequencies from the formulas; an entry is off by half a unit of 2^-64 and by what 64-bit logarithms and powers here lose."""
    theta = 500000.0
    if kind == "ntk" and rot == 2:
        pytest.skip("refused")
    got, magnitude = lc.rope_turns_scaled(theta, rot, kind, factor, original)
    if kind == "none":
        assert (got == lc.rope_turns(theta, rot)).all() and magnitude == 1.0
    base = theta * factor ** (rot / (rot - 2)) if kind == "ntk" and rot else theta
    f = np.array([base ** (-2.0 * d / rot) for d in range(rot // 2)])
    if kind == "linear":
        f = f / factor
    elif kind == "llama3":
        keep = np.clip((original * f / (2 * math.pi) - 1) / 3, 0, 1)
        f = keep * f + (1 - keep) * f / factor
    elif kind == "yarn":
        pair = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - low) / max(high - low, 0.001), 0, 1)
        f = f * (1 - ramp) + f / factor * ramp
    want = f / (2 * math.pi) * 2.0 ** 64
    assert np.abs(got.astype(np.float64) - want).max(initial=0.0) <= 2.0 ** -46 * want.max(initial=0.0) + 1
    assert abs(magnitude - (0.1 * math.log(factor) + 1 if kind == "yarn" else 1.0)) < 1e-15
