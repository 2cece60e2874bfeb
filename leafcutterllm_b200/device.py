"""Operators on tensors that are already on the GPU: rotary positions, the key/value caches in 8 and in 4 bits, and log probabilities.

The counterparts of the `_dev` calls of include/leafcutter_b200.h for torch tensors.  A call queues its kernels on torch's current
stream of the tensors' device (or on `stream`: a torch stream or a cudaStream_t as an integer) and returns without waiting; it allocates nothing but
what it is not given, from torch's allocator and as that stream's memory (a stream given as a number: nothing), so it can be captured into a graph.  Shapes, types and devices are checked
here, everything else by the library (LeafcutterError).  Nothing of the reference's corresponds to them.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _capi
from ._capi import TYPE_BF16, TYPE_F16, TYPE_F32, Kv4CacheStruct, Kv8CacheStruct, Kv8RowsStruct, check, load

_TYPES = {}
_raw_stream = None


def _torch():
    global _raw_stream
    import torch
    if not _TYPES:
        _TYPES.update({torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16})
        # the handle of the current stream alone, where torch has a way to it: making a stream object costs 2 us
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
    return torch


def _stream(index, stream):
    """A cudaStream_t: the current stream of device `index` where none is given.  Handle 0 is the legacy stream there; the library takes 0 for its own."""
    handle = _raw_stream(index) if stream is None else getattr(stream, "cuda_stream", stream)
    return handle or 1  # cudaStreamLegacy


def _empty(call, like, shape, dtype, stream):
    """A tensor on the device of `like`, from the memory of the stream that will write it: the current stream's may still be at work on what it frees."""
    torch = _torch()
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    if not hasattr(stream, "cuda_stream"):
        raise ValueError(f"{call}: a stream given as a number needs outputs and workspaces of the caller's")
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=like.device)


def _typ(t):
    if not _TYPES:
        _torch()
    typ = _TYPES.get(t.dtype)
    if typ is None:
        raise ValueError(f"{t.dtype}: float32, float16 and bfloat16 are taken")
    return typ


def _elsewhere(index, *tensors):
    raise ValueError(f"tensors on one device expected: {['cuda:%d' % index if index >= 0 else 'cpu'] + [str(t.device) for t in tensors if t is not None]}")


def _rows(t, heads, dim, what):
    """Rows [n][heads][dim] whose heads and dims are contiguous: the distance between rows, in elements."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what}: [rows, {heads if heads is not None else 'heads'}, {dim}] expected, got {list(shape)}")
    if t.is_contiguous():
        return shape[1] * dim
    stride = t.stride()
    if shape[0] and (stride[2] != 1 or (shape[1] > 1 and stride[1] != dim)):
        raise ValueError(f"{what}: the heads of a row must be contiguous")
    return stride[0] if shape[0] > 1 else shape[1] * dim


def _contiguous(what, dtype, *tensors):
    for t in tensors:
        if t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{what}: contiguous tensors of {dtype} expected, got {t.dtype}")


def rope_turns(theta: float, rot_dim: int) -> np.ndarray:
    """The rotation table of Kv8Cache.append: uint64 [rot_dim / 2], fractions of a turn per position in units of 2^-64.  Put it on the GPU as
    int64 (`torch.from_numpy(turns.view("int64")).cuda()`)."""
    out = np.empty(max(rot_dim, 0) // 2, np.uint64)
    check(load().lc_rope_turns(float(theta), rot_dim, out.ctypes.data_as(C.c_void_p)))
    return out


class Kv8Rows:
    """Which positions of which sequences the rows of a call are: row r of sequence i stands at position ctx[i] + r - row_start[i] and lies
    on page page_table[i, position // page_tokens].  int32 tensors on the GPU, read when the kernels run: page_table
    [n_seqs, width], ctx [n_seqs], row_start [n_seqs + 1].  max_rows: the most rows that a sequence is expected to have (it chooses kernels,
    not results).  status: an int32 tensor of one element that a call raises to i + 1 where sequence i cannot be served, or None."""

    def __init__(self, page_table, ctx, row_start, max_rows: int, status=None):
        torch = _torch()
        n = ctx.shape[0]
        if page_table.dim() != 2 or page_table.shape[0] != n or ctx.dim() != 1 or tuple(row_start.shape) != (n + 1,):
            raise ValueError("Kv8Rows: page_table [n, width], ctx [n] and row_start [n + 1] expected")
        _contiguous("Kv8Rows", torch.int32, page_table, ctx, row_start)
        if status is not None:
            _contiguous("Kv8Rows", torch.int32, status)
            if status.numel() < 1:
                raise ValueError("Kv8Rows: status has no element")
        self.index = page_table.get_device()
        if ctx.get_device() != self.index or row_start.get_device() != self.index or (status is not None and status.get_device() != self.index):
            _elsewhere(self.index, ctx, row_start, status)
        self._kept = (page_table, ctx, row_start, status)
        self.struct = Kv8RowsStruct(page_table.data_ptr(), ctx.data_ptr(), row_start.data_ptr(), status.data_ptr() if status is not None else None,
                                    n, page_table.shape[1], max_rows, 0)
        self._ref = C.addressof(self.struct)


class Kv8Cache:
    """A key/value cache in 8 bits: k and v int8 [pages, kv heads, page_tokens, head_dim], k_scale and v_scale float32 [pages, kv heads]; a cached
    element is its integer times the scale of its page and head.  page_tokens is 16, 32, 64, 128 or 256, head_dim a multiple of 16, at most 256."""

    def __init__(self, k, v, k_scale, v_scale):
        torch = _torch()
        if k.dim() != 4 or v.shape != k.shape or k_scale.shape != k.shape[:2] or v_scale.shape != k.shape[:2]:
            raise ValueError("Kv8Cache: k and v [pages, kv heads, page_tokens, head_dim], scales [pages, kv heads] expected")
        _contiguous("Kv8Cache", torch.int8, k, v)
        _contiguous("Kv8Cache", torch.float32, k_scale, v_scale)
        self.device, self.index = k.device, k.get_device()
        if v.get_device() != self.index or k_scale.get_device() != self.index or v_scale.get_device() != self.index:
            _elsewhere(self.index, v, k_scale, v_scale)
        self._kept = (k, v, k_scale, v_scale)
        self.n_kv_heads, self.page_tokens, self.head_dim = k.shape[1:]
        self.struct = Kv8CacheStruct(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.shape)
        self._ref = C.addressof(self.struct)

    def append(self, rows: Kv8Rows, k, v, turns=None, q=None, q_out=None, stream=None):
        """Appends rows of keys and values [rows, kv heads, head_dim] at their positions, the keys rotated by `turns` (rope_turns on the GPU; None: not
        rotated), q [rows, heads, head_dim] likewise into q_out (None: a new tensor; it may be q).  Returns q_out.  A page that receives rows
        must belong to one sequence of the call."""
        typ, n, index = _typ(k), k.shape[0], self.index
        if v.dtype != k.dtype or v.shape[0] != n:
            raise ValueError("append: keys and values of one type and as many rows expected")
        ks, vs = _rows(k, self.n_kv_heads, self.head_dim, "k"), _rows(v, self.n_kv_heads, self.head_dim, "v")
        if rows.index != index or k.get_device() != index or v.get_device() != index:
            _elsewhere(index, k, v)
        qp = qs = op = os = heads = tp = rot = 0
        if q is not None:
            if q_out is None:
                q_out = _empty("append", q, q.shape, q.dtype, stream)
            heads = q.shape[1]
            if q.dtype != k.dtype or q_out.dtype != k.dtype or q.shape[0] != n or q_out.shape[0] != n:
                raise ValueError("append: queries of the keys' type and as many rows expected, q_out like q")
            qs, os = _rows(q, None, self.head_dim, "q"), _rows(q_out, heads, self.head_dim, "q_out")
            qp, op = q.data_ptr(), q_out.data_ptr()
            if q.get_device() != index or q_out.get_device() != index:
                _elsewhere(index, q, q_out)
        if turns is not None:
            if turns.element_size() != 8 or turns.is_floating_point() or turns.is_complex() or not turns.is_contiguous() or turns.dim() != 1:
                raise ValueError("append: turns are contiguous 64-bit integers")
            if turns.get_device() != index:
                _elsewhere(index, turns)
            tp, rot = turns.data_ptr(), 2 * turns.shape[0]
        check(load().lc_kv8_append_dev(self._ref, rows._ref, typ, n, k.data_ptr(), ks, v.data_ptr(), vs, qp, qs, op, os, heads, tp, rot,
                                       _stream(index, stream)))
        return q_out

    def read(self, rows: Kv8Rows, k_out=None, v_out=None, stream=None):
        """The cached rows as values, into k_out and v_out [rows, kv heads, head_dim] (either may be None)."""
        some = k_out if k_out is not None else v_out
        if some is None:
            raise ValueError("read: nothing to read into")
        typ = _typ(some)
        if rows.index != self.index or some.get_device() != self.index or (v_out is not None and v_out.get_device() != self.index):
            _elsewhere(self.index, k_out, v_out)
        p, s = [0, 0], [0, 0]
        for i, t in enumerate((k_out, v_out)):
            if t is not None:
                if t.dtype != some.dtype or t.shape[0] != some.shape[0]:
                    raise ValueError("read: k_out and v_out of one type and as many rows expected")
                p[i], s[i] = t.data_ptr(), _rows(t, self.n_kv_heads, self.head_dim, "k_out" if i == 0 else "v_out")
        check(load().lc_kv8_read_dev(self._ref, rows._ref, typ, some.shape[0], p[0], s[0], p[1], s[1], _stream(self.index, stream)))
        return k_out, v_out

    def attention_workspace(self, rows: Kv8Rows, q) -> int:
        """Bytes of workspace of attention over such rows, or over fewer: no more rows, sequences, pages and max_rows than these."""
        typ = _typ(q)
        out = C.c_size_t()
        check(load().lc_attention_kv8_workspace(self._ref, rows._ref, typ, q.shape[0], q.shape[1], C.byref(out)))
        return int(out.value)

    def attention(self, rows: Kv8Rows, q, out=None, scale: float = None, window: int = 0, workspace=None, stream=None):
        """Attention of q [rows, heads, head_dim], already rotated, over the cache: each row attends to the positions up to its own (with
        window > 0 to the last `window` of them), which the cache already holds.  scale None: 1 / sqrt(head_dim).  Returns out.  workspace: a uint8 tensor of
        attention_workspace bytes (None: a new one); calls that may run at the same time need one each."""
        typ, index = _typ(q), self.index
        qs = _rows(q, None, self.head_dim, "q")
        n, heads = q.shape[:2]
        if out is None:
            out = _empty("attention", q, q.shape, q.dtype, stream)
        if out.dtype != q.dtype or out.shape[0] != n:
            raise ValueError("attention: out like q expected")
        os = _rows(out, heads, self.head_dim, "out")
        if workspace is None:
            workspace = _empty("attention", q, self.attention_workspace(rows, q), _torch().uint8, stream)
        elif not workspace.is_contiguous():
            raise ValueError("attention: a contiguous workspace expected")
        if rows.index != index or q.get_device() != index or out.get_device() != index or workspace.get_device() != index:
            _elsewhere(index, q, out, workspace)
        check(load().lc_attention_kv8_dev(self._ref, rows._ref, typ, n, q.data_ptr(), qs, heads, 0.0 if scale is None else scale, min(window, 2 ** 31 - 1), out.data_ptr(), os,
                                          workspace.data_ptr(), workspace.nbytes, _stream(index, stream)))
        return out


_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "llama3": 4}


def _layout(layout):
    number = _LAYOUTS.get(layout)
    if number is None:
        raise ValueError(f"layout {layout!r}: one of {sorted(_LAYOUTS)}")
    return number


def _turns(call, turns, index):
    """Pointer and rotated dims of a table on the GPU"""
    if turns.element_size() != 8 or turns.is_floating_point() or turns.is_complex() or turns.dim() != 1 or not turns.is_contiguous():
        raise ValueError(f"{call}: turns are contiguous 64-bit integers")
    if turns.get_device() != index:
        _elsewhere(index, turns)
    return turns.data_ptr(), 2 * turns.numel()


def rope_turns_scaled(theta: float, rot_dim: int, scaling: str = "none", factor: float = 1.0, original: int = 0, fast: float = 0.0, slow: float = 0.0):
    """(table, magnitude) for contexts `factor` times as long as the `original` one: the rotation table as of rope_turns, and what turned values are multiplied by.
    scaling: none; linear (all frequencies divided by factor); ntk (the base raised); yarn and llama3 (pairs of fewer than `slow` turns within the original
    length divided by factor, those of more than `fast` as they are, the others mixed; yarn has a magnitude above 1).  fast and slow of 0: the usual ones."""
    if scaling not in _SCALINGS:
        raise ValueError(f"scaling {scaling!r}: one of {sorted(_SCALINGS)}")
    out, magnitude = np.empty(max(rot_dim, 0) // 2, np.uint64), C.c_double()
    check(load().lc_rope_turns_scaled(float(theta), rot_dim, _SCALINGS[scaling], float(factor), original, float(fast), float(slow), out.ctypes.data_as(C.c_void_p), C.byref(magnitude)))
    return out, magnitude.value


def rope_dev(x, positions, turns, layout: str = "half", magnitude: float = 1.0, inverse: bool = False, out=None, y=None, y_out=None, stream=None):
    """Rows of heads x [rows, heads, dim] turned by their positions (int64 [rows]): of each head the first 2 * len(turns) dims, pairs (d, d + half of them) or, interleaved,
    (2 d, 2 d + 1), times `magnitude`; the others are copied.  inverse: the other way round, which is also the way of gradients.  y: a second tensor of the same
    rows.  Outputs that are None are made; they may be the inputs.  Returns out, or (out, y_out) where y is given."""
    typ, index, shape, dtype = _typ(x), x.get_device(), x.shape, x.dtype
    n, dim = shape[0], shape[-1]
    xs = _rows(x, None, dim, "x")
    heads = shape[1]
    if out is None:
        out = _empty("rope_dev", x, shape, dtype, stream)
    if positions.dtype != _torch().int64 or positions.dim() != 1 or positions.shape[0] != n or not positions.is_contiguous():
        raise ValueError("rope_dev: one position per row expected, contiguous int64")
    tp, rot = _turns("rope_dev", turns, index)
    yp = ys = op = os = yh = 0
    if y is not None:
        if y_out is None:
            y_out = _empty("rope_dev", y, y.shape, y.dtype, stream)
        ys, yh = _rows(y, None, dim, "y"), y.shape[1]
        os = _rows(y_out, yh, dim, "y_out")
        if y.dtype != dtype or y_out.dtype != dtype or y.shape[0] != n or y_out.shape[0] != n:
            raise ValueError("rope_dev: y of x's type and as many rows expected, y_out like y")
        yp, op = y.data_ptr(), y_out.data_ptr()
        if y.get_device() != index or y_out.get_device() != index:
            _elsewhere(index, y, y_out)
    if out.dtype != dtype or out.shape[0] != n:
        raise ValueError("rope_dev: out like x expected")
    if positions.get_device() != index or out.get_device() != index:
        _elsewhere(index, positions, out)
    check(load().lc_rope_dev(typ, n, positions.data_ptr(), tp, rot, dim, _layout(layout), 1 if inverse else 0, magnitude, x.data_ptr(), xs, out.data_ptr(), _rows(out, heads, dim, "out"), heads,
                             yp, ys, op, os, yh, _stream(index, stream)))
    return out if y is None else (out, y_out)


class Kv4Cache:
    """A key/value cache in 4 bits: k and v uint8 [pages, kv heads, page_tokens, head_dim / 2], two integers from -7 to 7 in a byte (as n + 8, the even dim low); k_block and v_block uint8
    [pages, kv heads, page_tokens, head_dim / 16], a scale in e4m3 for 16 dims of a row; k_scale and v_scale float32 [kv heads], positive.  A value is the product of the three; up to
    3136 times the head's scale is held.  page_tokens and head_dim as of Kv8Cache.  Its rows are Kv8Rows; a row lies in a slot, and its position may be another number."""

    def __init__(self, k, v, k_block, v_block, k_scale, v_scale):
        torch = _torch()
        if k.dim() != 4 or v.shape != k.shape or k.shape[3] % 8 or k_block.shape != (*k.shape[:3], k.shape[3] // 8) or v_block.shape != k_block.shape or k_scale.shape != k.shape[1:2] or v_scale.shape != k.shape[1:2]:
            raise ValueError("Kv4Cache: k and v [pages, kv heads, page_tokens, head_dim / 2], blocks [pages, kv heads, page_tokens, head_dim / 16], scales [kv heads] expected")
        _contiguous("Kv4Cache", torch.uint8, k, v, k_block, v_block)
        _contiguous("Kv4Cache", torch.float32, k_scale, v_scale)
        self.device, self.index = k.device, k.get_device()
        for t in (v, k_block, v_block, k_scale, v_scale):
            if t.get_device() != self.index:
                _elsewhere(self.index, v, k_block, v_block, k_scale, v_scale)
        self._kept = (k, v, k_block, v_block, k_scale, v_scale)
        self.n_kv_heads, self.page_tokens, self.head_dim = k.shape[1], k.shape[2], 2 * k.shape[3]
        self.struct = Kv4CacheStruct(k.data_ptr(), v.data_ptr(), k_block.data_ptr(), v_block.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.shape[:3], self.head_dim)
        self._ref = C.addressof(self.struct)

    def append(self, rows: Kv8Rows, k, v, turns=None, q=None, q_out=None, positions=None, layout: str = "half", magnitude: float = 1.0, stream=None):
        """Appends rows of keys and values [rows, kv heads, head_dim] in their slots, the keys turned by `turns` (rope_turns on the GPU; None: not turned), q [rows,
        heads, head_dim] likewise into q_out (None: a new tensor; it may be q).  positions: int64 [n_seqs], of each sequence's first row (None: its slot); layout and magnitude as of
        rope_dev.  Returns q_out.  A page that receives rows must belong to one sequence of the call."""
        typ, n, index = _typ(k), k.shape[0], self.index
        if v.dtype != k.dtype or v.shape[0] != n:
            raise ValueError("append: keys and values of one type and as many rows expected")
        ks, vs = _rows(k, self.n_kv_heads, self.head_dim, "k"), _rows(v, self.n_kv_heads, self.head_dim, "v")
        if rows.index != index or k.get_device() != index or v.get_device() != index:
            _elsewhere(index, k, v)
        qp = qs = op = os = heads = tp = rot = pp = 0
        if q is not None:
            if q_out is None:
                q_out = _empty("append", q, q.shape, q.dtype, stream)
            heads = q.shape[1]
            if q.dtype != k.dtype or q_out.dtype != k.dtype or q.shape[0] != n or q_out.shape[0] != n:
                raise ValueError("append: queries of the keys' type and as many rows expected, q_out like q")
            qs, os = _rows(q, None, self.head_dim, "q"), _rows(q_out, heads, self.head_dim, "q_out")
            qp, op = q.data_ptr(), q_out.data_ptr()
            if q.get_device() != index or q_out.get_device() != index:
                _elsewhere(index, q, q_out)
        if turns is not None:
            tp, rot = _turns("append", turns, index)
        if positions is not None:
            _contiguous("append", _torch().int64, positions)
            if tuple(positions.shape) != (rows.struct.n_seqs,):
                raise ValueError("append: one position per sequence expected")
            if positions.get_device() != index:
                _elsewhere(index, positions)
            pp = positions.data_ptr()
        check(load().lc_kv4_append_dev(self._ref, rows._ref, typ, n, pp, k.data_ptr(), ks, v.data_ptr(), vs, qp, qs, op, os, heads, tp, rot, _layout(layout), magnitude, _stream(index, stream)))
        return q_out

    def read(self, rows: Kv8Rows, k_out=None, v_out=None, stream=None):
        """The cached rows as values, into k_out and v_out [rows, kv heads, head_dim] (either may be None)."""
        some = k_out if k_out is not None else v_out
        if some is None:
            raise ValueError("read: nothing to read into")
        typ = _typ(some)
        if rows.index != self.index or some.get_device() != self.index or (v_out is not None and v_out.get_device() != self.index):
            _elsewhere(self.index, k_out, v_out)
        p, s = [0, 0], [0, 0]
        for i, t in enumerate((k_out, v_out)):
            if t is not None:
                if t.dtype != some.dtype or t.shape[0] != some.shape[0]:
                    raise ValueError("read: k_out and v_out of one type and as many rows expected")
                p[i], s[i] = t.data_ptr(), _rows(t, self.n_kv_heads, self.head_dim, "k_out" if i == 0 else "v_out")
        check(load().lc_kv4_read_dev(self._ref, rows._ref, typ, some.shape[0], p[0], s[0], p[1], s[1], _stream(self.index, stream)))
        return k_out, v_out

    def attention_workspace(self, rows: Kv8Rows, q) -> int:
        """Bytes of workspace of attention over such rows, or over fewer: no more rows, sequences, pages and max_rows than these."""
        out = C.c_size_t()
        check(load().lc_attention_kv4_workspace(self._ref, rows._ref, _typ(q), q.shape[0], q.shape[1], C.byref(out)))
        return int(out.value)

    def _lse(self, call, lse, n, heads):
        if lse.dtype != _torch().float32 or tuple(lse.shape) != (n, heads) or (heads > 1 and lse.stride(1) != 1):
            raise ValueError(f"{call}: lse is float32 [rows, heads], the heads contiguous")
        if lse.get_device() != self.index:
            _elsewhere(self.index, lse)
        return lse.data_ptr(), lse.stride(0) if n > 1 else heads

    def attention(self, rows: Kv8Rows, q, out=None, lse=None, scale: float = None, window: int = 0, workspace=None, stream=None):
        """Attention of q [rows, heads, head_dim], already turned, over the cache: each row attends to the slots up to its own (with window > 0 to the last
        `window` of them), which the cache already holds.  scale None (or 0): 1 / sqrt(head_dim).  Returns out.  lse: float32 [rows, heads], which receives ln sum exp of the scores.  workspace: a uint8 tensor of
        attention_workspace bytes (None: a new one); calls that may run at the same time need one each."""
        typ, index = _typ(q), self.index
        qs = _rows(q, None, self.head_dim, "q")
        n, heads = q.shape[:2]
        if out is None:
            out = _empty("attention", q, q.shape, q.dtype, stream)
        if out.dtype != q.dtype or out.shape[0] != n:
            raise ValueError("attention: out like q expected")
        os = _rows(out, heads, self.head_dim, "out")
        lp, ls = (0, 0) if lse is None else self._lse("attention", lse, n, heads)
        if workspace is None:
            workspace = _empty("attention", q, self.attention_workspace(rows, q), _torch().uint8, stream)
        elif not workspace.is_contiguous():
            raise ValueError("attention: a contiguous workspace expected")
        if rows.index != index or q.get_device() != index or out.get_device() != index or workspace.get_device() != index:
            _elsewhere(index, q, out, workspace)
        check(load().lc_attention_kv4_dev(self._ref, rows._ref, typ, n, q.data_ptr(), qs, heads, 0.0 if scale is None else scale, min(window, 2 ** 31 - 1), out.data_ptr(), os, lp, ls,
                                          workspace.data_ptr(), workspace.nbytes, _stream(index, stream)))
        return out

    def _mass(self, call, rows, mass):
        """float32 [n_seqs, kv heads, capacity], the last dim contiguous: pointer, strides, capacity"""
        if mass.dtype != _torch().float32 or mass.dim() != 3 or tuple(mass.shape[:2]) != (rows.struct.n_seqs, self.n_kv_heads) or (mass.shape[2] > 1 and mass.stride(2) != 1):
            raise ValueError(f"{call}: mass is float32 [n_seqs, {self.n_kv_heads}, capacity], the slots contiguous")
        if mass.get_device() != self.index or rows.index != self.index:
            _elsewhere(self.index, mass)
        cap = mass.shape[2]
        return mass.data_ptr(), mass.stride(0) if mass.shape[0] > 1 else max(cap, mass.stride(0)), mass.stride(1) if mass.shape[1] > 1 else cap, cap

    def weights(self, rows: Kv8Rows, q, lse, mass, scale: float = None, window: int = 0, stream=None):
        """Adds to mass (float32 [n_seqs, kv heads, capacity]) what weight the rows gave each cached key, summed over the rows and the heads of a group; q and lse as attention over these
        rows had and gave them.  A caller may take some rows only (the last ones of a prompt).  Returns mass."""
        typ, index = _typ(q), self.index
        qs = _rows(q, None, self.head_dim, "q")
        n, heads = q.shape[:2]
        lp, ls = self._lse("weights", lse, n, heads)
        mp, ms, mh, cap = self._mass("weights", rows, mass)
        if q.get_device() != index:
            _elsewhere(index, q)
        check(load().lc_kv4_weights_dev(self._ref, rows._ref, typ, n, q.data_ptr(), qs, heads, 0.0 if scale is None else scale, min(window, 2 ** 31 - 1), lp, ls, mp, ms, mh, cap, _stream(index, stream)))
        return mass

    def evict(self, rows: Kv8Rows, mass, keep: int, limit: int = None, recent: int = 0, first: int = 0, kept=None, ctx_out=None, stream=None):
        """Cuts sequences that hold more than `limit` rows (None: keep), their context and the call's rows, to `keep`: for each kv head the `first` first, the `recent` last and the heaviest between
        move to the front, in their order, and their sums in mass with them.  Returns (kept int32 [n_seqs, kv heads, limit], the slots that they came from, -1 behind them; ctx_out int32 [n_seqs], the new
        lengths).  The pages of a sequence that is cut must be its own.  Fastest where mass's capacity is not far above limit and a call's rows."""
        torch, index, n = _torch(), self.index, rows.struct.n_seqs
        limit = keep if limit is None else limit
        mp, ms, mh, cap = self._mass("evict", rows, mass)
        if kept is None:
            kept = _empty("evict", mass, (n, self.n_kv_heads, max(limit, 0)), torch.int32, stream)
        if ctx_out is None:
            ctx_out = _empty("evict", mass, (n,), torch.int32, stream)
        _contiguous("evict", torch.int32, kept, ctx_out)
        if tuple(kept.shape) != (n, self.n_kv_heads, max(limit, 0)) or tuple(ctx_out.shape) != (n,):
            raise ValueError(f"evict: kept [n_seqs, {self.n_kv_heads}, {limit}] and ctx_out [n_seqs] expected")
        if kept.get_device() != index or ctx_out.get_device() != index:
            _elsewhere(index, kept, ctx_out)
        check(load().lc_kv4_evict_dev(self._ref, rows._ref, mp, ms, mh, cap, keep, limit, recent, first, kept.data_ptr(), ctx_out.data_ptr(), _stream(index, stream)))
        return kept, ctx_out


def token_logprobs_dev(logits, tokens, logprob=None, entropy=None, top_logprob=None, top_id=None, top: int = None, stream=None):
    """Log probabilities of `tokens` (int64 [rows]) under logits [rows, vocab], entropies of the rows (nats), and the `top` likeliest tokens with theirs
    (larger logit first, equal ones by the lower index).  Outputs that are None are made; `top` (0 .. 32) is the width of
    top_id where that is given, else 0 unless said.  Returns (logprob, entropy, top_logprob, top_id)."""
    typ, index = _typ(logits), logits.get_device()
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 2 or (shape[0] and shape[1] > 1 and stride[1] != 1):
        raise ValueError("token_logprobs_dev: logits [rows, vocab] with contiguous rows expected")
    rows, vocab = shape
    torch = _torch()
    if (top_logprob is None) != (top_id is None):
        raise ValueError("token_logprobs_dev: top_logprob and top_id go together")
    if top_id is not None and top is not None and top_id.shape[-1] != top:
        raise ValueError("token_logprobs_dev: top_id is not `top` wide")
    top = top_id.shape[-1] if top_id is not None else top or 0
    if logprob is None:
        logprob = _empty("token_logprobs_dev", logits, rows, torch.float32, stream)
    if entropy is None:
        entropy = _empty("token_logprobs_dev", logits, rows, torch.float32, stream)
    if top_id is None:
        top_logprob = _empty("token_logprobs_dev", logits, (rows, max(top, 0)), torch.float32, stream)
        top_id = _empty("token_logprobs_dev", logits, (rows, max(top, 0)), torch.int64, stream)
    _contiguous("token_logprobs_dev", torch.int64, tokens, top_id)
    _contiguous("token_logprobs_dev", torch.float32, logprob, entropy, top_logprob)
    one, wide = (rows,), (rows, top)
    if tokens.shape != one or logprob.shape != one or entropy.shape != one or top_logprob.shape != wide or top_id.shape != wide:
        raise ValueError("token_logprobs_dev: one token and one output per row expected")
    if any(t.get_device() != index for t in (tokens, logprob, entropy, top_logprob, top_id)):
        _elsewhere(index, tokens, logprob, entropy, top_logprob, top_id)
    check(load().lc_token_logprobs_dev(typ, logits.data_ptr(), rows, vocab, stride[0] if rows > 1 else vocab, tokens.data_ptr(), top, logprob.data_ptr(),
                                       entropy.data_ptr(), top_logprob.data_ptr(), top_id.data_ptr(), _stream(index, stream)))
    return logprob, entropy, top_logprob, top_id
