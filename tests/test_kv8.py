"""What the calls over the 8-bit key/value cache and of log probabilities refuse, and the rotation table: host code, no GPU.

Every refusal comes before the library looks for a device, so the pointers here are never read."""
import ctypes as C
import math

import numpy as np
import pytest

P = 1 << 20  # an address that is 16-byte aligned and never read
BF16, F32 = 30, 0


def cache(lc, **over):
    d = dict(k_dev=P, v_dev=P, k_scale_dev=P, v_scale_dev=P, n_pages=4, n_kv_heads=2, page_tokens=16, head_dim=64)
    d.update(over)
    return lc._capi.Kv8CacheStruct(**d)


def rows(lc, **over):
    d = dict(page_table_dev=P, ctx_dev=P, row_start_dev=P, status_dev=None, n_seqs=2, table_width=3, max_rows=1, reserved=0)
    d.update(over)
    return lc._capi.Kv8RowsStruct(**d)


def append(lc, c=None, r=None, typ=F32, n=2, k=P, ks=128, v=P, vs=128, q=None, qs=0, qo=None, os=0, heads=0, turns=P, rot=64):
    return lc.load().lc_kv8_append_dev(C.byref(c or cache(lc)), C.byref(r or rows(lc)), typ, n, k, ks, v, vs, q, qs, qo, os, heads, turns, rot, None)


def read(lc, c=None, r=None, typ=F32, n=2, k=P, ks=128, v=P, vs=128):
    return lc.load().lc_kv8_read_dev(C.byref(c or cache(lc)), C.byref(r or rows(lc)), typ, n, k, ks, v, vs, None)


def attend(lc, c=None, r=None, typ=F32, n=2, q=P, qs=256, heads=4, scale=0.0, window=0, out=P, os=256, ws=P, wb=1 << 40):
    return lc.load().lc_attention_kv8_dev(C.byref(c or cache(lc)), C.byref(r or rows(lc)), typ, n, q, qs, heads, scale, window, out, os, ws, wb, None)


BAD_CACHE = [dict(k_dev=None), dict(v_dev=None), dict(k_scale_dev=None), dict(v_scale_dev=None), dict(k_dev=P + 8), dict(v_dev=P + 1), dict(n_pages=0),
             dict(n_kv_heads=0), dict(n_kv_heads=1025), dict(head_dim=0), dict(head_dim=72), dict(head_dim=272), dict(page_tokens=0),
             dict(page_tokens=8), dict(page_tokens=24), dict(page_tokens=512)]
BAD_ROWS = [dict(n_seqs=-1), dict(n_seqs=4097), dict(table_width=-1), dict(table_width=1 << 30), dict(max_rows=-1), dict(page_table_dev=None),
            dict(ctx_dev=None), dict(row_start_dev=None)]


@pytest.mark.parametrize("call", [append, read, attend])
@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_caches_are_refused(lc, call, bad):
    assert call(lc, c=cache(lc, **bad)) == lc._capi.LC_ERR_INVALID
    assert lc.load().lc_last_error()


@pytest.mark.parametrize("call", [append, read, attend])
@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_bad_rows_are_refused(lc, call, bad):
    assert call(lc, r=rows(lc, **bad)) == lc._capi.LC_ERR_INVALID


@pytest.mark.parametrize("call", [append, read, attend])
def test_types_and_row_counts(lc, call):
    assert call(lc, typ=8) == lc._capi.LC_ERR_UNSUPPORTED
    assert call(lc, n=-1) == lc._capi.LC_ERR_INVALID
    assert call(lc, n=(1 << 24) + 1) == lc._capi.LC_ERR_INVALID
    assert call(lc, n=0) == lc._capi.LC_OK                          # nothing to do, even without a device
    assert call(lc, r=rows(lc, n_seqs=0)) == lc._capi.LC_OK


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(ks=127), dict(vs=0), dict(rot=63), dict(rot=66), dict(rot=-2), dict(turns=None),
                                 dict(q=P, qo=None, qs=256, os=256, heads=4), dict(q=P, qo=P, qs=255, os=256, heads=4),
                                 dict(q=P, qo=P, qs=256, os=255, heads=4), dict(q=P, qo=P, qs=256, os=256, heads=0)], ids=str)
def test_append_refuses(lc, bad):
    assert append(lc, **bad) == lc._capi.LC_ERR_INVALID


@pytest.mark.parametrize("bad", [dict(ks=127), dict(vs=127)], ids=str)
def test_read_refuses(lc, bad):
    assert read(lc, **bad) == lc._capi.LC_ERR_INVALID


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(qs=255), dict(os=1), dict(heads=0), dict(heads=3), dict(window=-1), dict(scale=-1.0),
                                 dict(scale=math.inf), dict(scale=math.nan)], ids=str)
def test_attention_refuses(lc, bad):
    assert attend(lc, **bad) == lc._capi.LC_ERR_INVALID


def test_attention_refuses_what_its_counters_cannot_hold(lc):
    wide = rows(lc, table_width=1 << 24, n_seqs=4096)
    assert attend(lc, r=wide, n=1 << 20, heads=64) == lc._capi.LC_ERR_INVALID


def logprobs_dev(lc, typ=F32, x=P, n=2, vocab=100, stride=100, tokens=P, top=3, lp=P, ent=P, tl=P, ti=P):
    return lc.load().lc_token_logprobs_dev(typ, x, n, vocab, stride, tokens, top, lp, ent, tl, ti, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(n=-1), dict(vocab=0), dict(vocab=101), dict(stride=99), dict(top=-1), dict(top=33), dict(vocab=2, top=3),
                                 dict(tokens=None), dict(tl=None), dict(ti=None)], ids=str)
def test_logprobs_refuse(lc, bad):
    assert logprobs_dev(lc, **bad) == lc._capi.LC_ERR_INVALID


def test_logprobs_types(lc):
    assert logprobs_dev(lc, typ=12) == lc._capi.LC_ERR_UNSUPPORTED
    assert logprobs_dev(lc, n=0) == lc._capi.LC_OK


def test_host_logprobs_refuse(lc):
    x = np.zeros((2, 10), np.float32)
    for bad in (dict(top=11), dict(top=-1), dict(top=33)):
        with pytest.raises(lc.LeafcutterError):
            lc.token_logprobs(x, [0, 1], **bad)
    with pytest.raises(ValueError):
        lc.token_logprobs(x, [0])
    with pytest.raises(ValueError):
        lc.token_logprobs(x[0], [0])


def test_no_device_is_an_error(lc):
    if lc.load().lc_device_count() > 0:
        pytest.skip("a device is present")
    assert append(lc) == read(lc) == attend(lc) == logprobs_dev(lc) == lc._capi.LC_ERR_CUDA


def test_turns(lc):
    for theta, dim in ((10000.0, 128), (500000.0, 64), (1.0, 2), (10000.0, 0)):
        got = lc.rope_turns(theta, dim)
        assert got.shape == (dim // 2,) and got.dtype == np.uint64
        for d, g in enumerate(got):
            want = theta ** (-2.0 * d / dim) / (2 * math.pi)
            # an entry is a whole number of units of 2^-64, so at most half of one, 2^-65, off; the rest is the comparison's own arithmetic
            assert abs(int(g) / 2.0 ** 64 - want) <= 2.0 ** -65 + 4 * 2.0 ** -53 * want
    for bad in (dict(theta=0.5, rot_dim=64), dict(theta=math.inf, rot_dim=64), dict(theta=math.nan, rot_dim=64), dict(theta=10000.0, rot_dim=63), dict(theta=10000.0, rot_dim=-2)):
        with pytest.raises(lc.LeafcutterError):
            lc.rope_turns(**bad)


def test_tensors_of_other_kinds_are_refused(lc):
    import torch
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    s = torch.zeros(4, 2)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        lc.Kv8Cache(k.float(), k, s, s)
    with pytest.raises(ValueError):
        lc.Kv8Cache(k, k, s[:3], s)
    with pytest.raises(ValueError):
        lc.Kv8Cache(k.transpose(1, 2), k.transpose(1, 2), s, s)
    with pytest.raises(ValueError):
        lc.Kv8Rows(torch.zeros(2, 3, dtype=torch.int64), i32(0, 0), i32(0, 1, 2), 1)
    with pytest.raises(ValueError):
        lc.Kv8Rows(torch.zeros(2, 3, dtype=torch.int32), i32(0, 0), i32(0, 1), 1)
    c = lc.Kv8Cache(k, k, s, s)
    r = lc.Kv8Rows(torch.zeros(2, 3, dtype=torch.int32), i32(0, 0), i32(0, 1, 2), 1)
    x = torch.zeros(2, 2, 64)
    for kw in (dict(k=x.to(torch.int32), v=x), dict(k=x, v=x.half()), dict(k=x[:, :1], v=x), dict(k=x, v=x[:1]), dict(k=x, v=x.transpose(1, 2).contiguous().transpose(1, 2)),
               dict(k=x, v=x, q=torch.zeros(3, 4, 64)), dict(k=x, v=x, turns=torch.zeros(32))):
        with pytest.raises(ValueError):
            c.append(r, **kw)
    with pytest.raises(ValueError):
        c.read(r)
    with pytest.raises(ValueError):
        c.attention(r, torch.zeros(2, 4, 64), out=torch.zeros(2, 4, 64, dtype=torch.float16))
    with pytest.raises(ValueError):
        lc.token_logprobs_dev(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        lc.token_logprobs_dev(torch.zeros(2, 10), torch.zeros(3, dtype=torch.int64))
