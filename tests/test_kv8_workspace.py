"""The workspace of attention over the 8-bit cache: what the host says without a device."""
import ctypes as C

import pytest

from test_kv8 import cache, rows


def workspace(lc, typ, n, heads, **over):
    out = C.c_size_t(1 << 60)
    rc = lc.load().lc_attention_kv8_workspace(C.byref(cache(lc)), C.byref(rows(lc, **over)), typ, n, heads, C.byref(out))
    return rc, out.value


@pytest.mark.parametrize("typ", [0, 1, 30])
@pytest.mark.parametrize("max_rows", [0, 1, 8, 16, 32, 100, 4000])
@pytest.mark.parametrize("heads", [2, 8, 64])
def test_of_calls_that_have_nothing_to_do(lc, typ, max_rows, heads):
    """A step without sequences or rows asks for no more than an allocator's smallest piece, and the call itself takes it, with or without a device."""
    for n_seqs, n in ((0, 0), (0, 5), (0, 4000), (2, 0), (4096, 0)):
        rc, size = workspace(lc, typ, n, heads, n_seqs=n_seqs, max_rows=max_rows)
        assert rc == lc._capi.LC_OK and size <= 512


def test_arguments_are_checked_all_the_same(lc):
    assert workspace(lc, 0, 0, 3)[0] == lc._capi.LC_ERR_INVALID
    assert workspace(lc, 8, 0, 2)[0] == lc._capi.LC_ERR_UNSUPPORTED
    assert workspace(lc, 0, 0, 2, max_rows=-1)[0] == lc._capi.LC_ERR_INVALID


def tensors():
    import torch
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return torch, torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2), torch.zeros(2, 3, dtype=torch.int32), i32(0, 0), i32(0, 1, 2)


def test_workspaces_with_gaps_are_refused(lc):
    """Bytes between a view's are not the call's."""
    torch, k, s, table, ctx, start = tensors()
    c, r = lc.Kv8Cache(k, k, s, s), lc.Kv8Rows(table, ctx, start, 1)
    with pytest.raises(ValueError, match="workspace"):
        c.attention(r, torch.zeros(2, 4, 64), workspace=torch.zeros(1 << 20, dtype=torch.uint8)[::2])


def test_rotation_tables_of_other_types_are_refused(lc):
    torch, k, s, table, ctx, start = tensors()
    c, r = lc.Kv8Cache(k, k, s, s), lc.Kv8Rows(table, ctx, start, 1)
    x = torch.zeros(2, 2, 64)
    for dtype in (torch.complex64, torch.float64, torch.int32):
        with pytest.raises(ValueError, match="turns"):
            c.append(r, x, x, turns=torch.zeros(32, dtype=dtype))


def test_windows_beyond_32_bits(lc, monkeypatch):
    """As wide as a table can be, not what is left of them in 32 bits."""
    torch, k, s, table, ctx, start = tensors()
    c, r = lc.Kv8Cache(k, k, s, s), lc.Kv8Rows(table, ctx, start, 1)
    seen = []

    class Library:
        def lc_attention_kv8_dev(self, *a):
            seen.append(a[8])
            return lc._capi.LC_OK
    import leafcutterllm_b200.device as device
    monkeypatch.setattr(device, "load", lambda: Library())
    device._torch()
    monkeypatch.setattr(device, "_raw_stream", lambda index: 0)
    q, ws = torch.zeros(2, 4, 64), torch.zeros(64, dtype=torch.uint8)
    for window in (0, 5, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1):
        c.attention(r, q, torch.empty_like(q), window=window, workspace=ws)
        assert seen[-1] == min(window, 2 ** 31 - 1)
    c.attention(r, q, torch.empty_like(q), window=-1, workspace=ws)
    assert seen[-1] == -1                                 # the library refuses it


def test_rows_times_heads_beyond_31_bits_are_refused(lc):
    """The kernels count a sequence's rows times the heads of a group in 32 bits: a sequence outside its table may have all rows, however few pages there are."""
    from test_kv8 import attend
    one = cache(lc, n_kv_heads=1, head_dim=16)
    few = rows(lc, n_seqs=1, table_width=1, max_rows=1)
    for heads, n in ((256, 1 << 24), (128, 1 << 24), (65536, 1 << 15)):
        args = dict(c=one, r=few, n=n, heads=heads, qs=heads * 16, os=heads * 16)
        assert attend(lc, **args) == lc._capi.LC_ERR_INVALID and b"too many" in lc.load().lc_last_error()
        out = C.c_size_t()
        assert lc.load().lc_attention_kv8_workspace(C.byref(one), C.byref(few), 30, n, heads, C.byref(out)) == lc._capi.LC_ERR_INVALID
        assert b"too many" in lc.load().lc_last_error()
