"""The paged KV cache in 4 bits: append, read-back and attention as operators.

``DecodeEngine(w, max_batch, kv_bits=4)`` decodes and serves from such a cache;
the functions here are its parts, for one layer's pool of any ``n_kv`` heads of
64 or 128 dims (``b2d_kv4_*`` in include/b2d.h, which states the format: groups
of 16 dims with a scale of 8 bits, 4.5 bits a value, and held values exact in
bf16 and fp16).  The reference has no cache below bf16.

All calls are asynchronous and stream-ordered.  ``stream``: a stream of the
pool's device instead of the current one; the caller keeps the inputs (or
records them on it) until it is done with them, and orders it behind what wrote
them.  New outputs come from that stream's memory.  A pool is the uint8 tensor of
``new_kv4_pool``; a block of it holds 16 positions; ``table`` int32
[n_seqs, blocks_per_seq] names the block of positions 16i.. of each sequence.
Entries are read only where a position needs them.  Bad entries, positions and
lengths seen by a kernel set ``status`` (an int32 tensor of one item, 0 at
first) and skip the access; ``check_status`` raises for it.
"""

from __future__ import annotations

import ctypes
import functools

import numpy as np
import torch

from . import _lib

PAGE_TOKENS = 16  # positions per block
_TYPES = {torch.float32: _lib.B2D_F32, torch.bfloat16: _lib.B2D_BF16, torch.float16: _lib.B2D_F16}


def _stream_on(stream, index) -> int:
    """The stream's handle, by default the current one of the device `index`."""
    return stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(index)


def _empty_like(t, stream, dtype=None) -> torch.Tensor:
    """A tensor from the stream's own memory (as torch's allocator keeps it)."""
    if stream is None:
        return torch.empty_like(t, dtype=dtype)
    with torch.cuda.stream(stream):
        return torch.empty_like(t, dtype=dtype)


def page_bytes(d_head: int) -> int:
    """Bytes that 16 positions of one kv head take."""
    return 18 * d_head


def new_kv4_pool(num_blocks: int, n_kv: int, d_head: int, device=None) -> torch.Tensor:
    """Zeroed pool of one layer: uint8 [num_blocks, n_kv, 18 * d_head]."""
    if num_blocks < 1 or n_kv < 1 or d_head not in (64, 128):
        raise ValueError("a 4-bit pool needs blocks, kv heads and heads of 64 or 128 dims")
    return torch.zeros(num_blocks, n_kv, page_bytes(d_head), dtype=torch.uint8, device=device or "cuda")


def check_status(status: torch.Tensor) -> None:
    """Raises for bad input that a kernel met (synchronises)."""
    word = int(status.item())
    if word:
        raise _lib.B2DError(_lib.B2D_ERR_DEVICE_INPUT, "device status", f"word 0x{word & 0xffffffff:x}")


def _ints(t, name, index, n):
    if t.dtype is not torch.int32 or t.shape != (n,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} items on the pool's device")
    return t.data_ptr()


def _cache(pool, table, status):
    """(the C cache, its device, blocks_per_seq, table rows, kv heads, dims)"""
    index = pool.get_device()
    if index < 0:
        raise ValueError("pool must be on a GPU")
    if pool.dtype is not torch.uint8 or pool.dim() != 3 or not pool.is_contiguous():
        raise ValueError("pool must be contiguous uint8 [num_blocks, n_kv, 18 * d_head] (see new_kv4_pool)")
    blocks, n_kv, size = pool.shape
    if size not in (1152, 2304) or n_kv < 1 or blocks < 1:
        raise ValueError("pool must hold heads of 64 or 128 dims: uint8 [num_blocks, n_kv, 18 * d_head]")
    if table.dtype is not torch.int32 or table.dim() != 2 or table.get_device() != index or not table.is_contiguous():
        raise ValueError("table must be a contiguous int32 [n_seqs, blocks_per_seq] tensor on the pool's device")
    rows, bps = table.shape
    if rows < 1 or bps < 1:
        raise ValueError("table must name a block")
    if status is not None and (status.dtype is not torch.int32 or status.get_device() != index or status.numel() != 1):
        raise ValueError("status must be an int32 tensor of one item on the pool's device")
    d = size // 18
    return (_lib.Kv4Cache(pool.data_ptr(), table.data_ptr(), None if status is None else status.data_ptr(), n_kv, d,
                          blocks, bps, rows, index), index, bps, rows, n_kv, d)


def _strides(t, name, index, shape, types):
    """(address, row stride, head stride) of a [rows, heads, d] tensor with
    contiguous dims and any row and head strides."""
    if t.shape != shape or t.dtype not in types or t.get_device() != index:
        raise ValueError(f"{name} must be a {list(shape)} tensor on the pool's device, of "
                         + " or ".join(map(str, types)))
    row, head, one = t.stride()
    if one != 1:
        raise ValueError(f"{name} must have contiguous dims")
    return t.data_ptr(), row, head


def _starts(x) -> np.ndarray:
    """Sorted addresses of the contiguous pieces (last dim) of x."""
    at = np.zeros(1, np.int64)
    for size, stride in zip(x.shape[:-1], x.stride()[:-1]):
        at = (at[:, None] + np.arange(size) * stride).reshape(-1)
    return np.sort(x.data_ptr() + at * x.element_size())


def _overlap(x, y) -> bool:
    """Whether tensors of any outer strides (contiguous in their last dim) share a byte."""
    if not x.numel() or not y.numel():
        return False
    xs, ys = x.element_size(), y.element_size()
    xp, yp, x_shape, y_shape, x_str, y_str = x.data_ptr(), y.data_ptr(), x.shape, y.shape, x.stride(), y.stride()
    if (yp >= xp + xs * sum([(n - 1) * s for n, s in zip(x_shape, x_str)], 1)
            or xp >= yp + ys * sum([(n - 1) * s for n, s in zip(y_shape, y_str)], 1)):
        return False
    # views of one buffer's rows, side by side
    row = xs * x_str[0]
    x_row, y_row = (e * sum([(n - 1) * s for n, s in zip(shape[1:], st[1:])], 1)
                    for e, shape, st in ((xs, x_shape, x_str), (ys, y_shape, y_str)))
    if row == ys * y_str[0] and row > 0:
        off = (yp - xp) % row
        if off >= x_row and off + y_row <= row:
            return False
    a, b = _starts(x), _starts(y)
    x_len, y_len = xs * x_shape[-1], ys * y_shape[-1]
    return bool((np.searchsorted(b, a + x_len, "left") > np.searchsorted(b, a - y_len, "right")).any())


def _same_place(x, y) -> bool:
    """Whether tensors of one shape and type have the same elements."""
    return x.data_ptr() == y.data_ptr() and all(n < 2 or s == t for n, s, t in zip(x.shape, x.stride(), y.stride()))


def _folded(x) -> bool:
    """Whether two elements of x share their place."""
    need = 1
    for stride, size in sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1):
        if stride < need:
            break
        need = stride * size
    else:
        return False
    return bool(x.numel()) and bool((np.diff(_starts(x)) < x.shape[-1] * x.element_size()).any())


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(index, n_kv, d, heads, n_seqs, max_rows, max_len) -> int:
    """Bytes of scratch that a call of these sizes needs (a function of them alone)."""
    room = (max_len + PAGE_TOKENS - 1) // PAGE_TOKENS or 1
    cache = _lib.Kv4Cache(16, 16, None, n_kv, d, 1, room, n_seqs, index)  # (addresses that the query does not read)
    query = _lib.Kv4Query(16, 16, 0, 0, 0, 0, 16, 16, _lib.B2D_F16, max(max_rows, n_seqs), heads, n_seqs, max_rows,
                          max_len, 1.0)
    need = ctypes.c_uint64()
    _lib.check(_lib.load().b2d_kv4_attention_scratch(ctypes.byref(cache), ctypes.byref(query), ctypes.byref(need)),
               "b2d_kv4_attention_scratch")
    return need.value


def kv4_append(pool, k, v, pos, table, *, seq=None, q=None, q_out=None, cos=None, sin=None, interleaved=False,
               status=None, stream=None):
    """Writes the rows ``k``, ``v`` [n, n_kv, d] (float32, bf16 or fp16) to the
    positions ``pos`` (int32 [n]; negative: skipped) of the sequences ``seq``
    (int32 [n] rows of ``table``; default: row i is sequence i), quantised to 4
    bits, ``k`` turned by its position's angles on the way.

    ``cos``, ``sin``: float32 [max_pos, r / 2], the first r dims of each head
    turn (pairs i, i + r / 2; with ``interleaved`` 2i, 2i + 1); None: no
    rotation.  ``q`` [n, heads, d] is turned alike into ``q_out`` (default: a
    new tensor; may be ``q``; a float32 ``q`` also into bf16 or fp16), which is
    returned.  Two rows of a call at one position leave bytes of both there."""
    c, dev, _, table_rows, n_kv, d = _cache(pool, table, status)
    n = pos.numel()
    shape = (n, n_kv, d)
    k_ptr, k_row, k_head = _strides(k, "k", dev, shape, _TYPES)
    v_ptr, v_row, v_head = _strides(v, "v", dev, shape, (k.dtype,))
    if seq is None and n > table_rows:
        raise ValueError("more rows than table rows need seq")
    heads = rotary = max_pos = q_row = q_head = o_row = o_head = 0
    q_ptr = o_ptr = None
    dtype = o_type = _TYPES[k.dtype]
    if q is not None:
        heads = q.shape[1] if q.dim() == 3 else 0
        q_ptr, q_row, q_head = _strides(q, "q", dev, (n, heads, d), (k.dtype,))
        if heads < 1:
            raise ValueError("q needs a head")
        given = q_out is not None
        if not given:
            q_out = _empty_like(q, stream)
        o_ptr, o_row, o_head = _strides(q_out, "q_out", dev, (n, heads, d),
                                        _TYPES if q.dtype is torch.float32 else (q.dtype,))
        o_type = _TYPES[q_out.dtype]
        if given and (_folded(q_out) or _overlap(q_out, k) or _overlap(q_out, v) or (
                not (o_type == dtype and _same_place(q_out, q)) and _overlap(q_out, q))):
            raise ValueError("q_out must be q or apart from it, and apart from k and v")
    elif q_out is not None:
        raise ValueError("q_out without q")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        max_pos, half = cos.shape if cos.dim() == 2 else (0, 0)
        rotary = 2 * half
        for t in (cos, sin):
            if t.dtype is not torch.float32 or t.shape != (max_pos, half) or t.get_device() != dev or (
                    not t.is_contiguous()) or not 2 <= rotary <= d or max_pos < 1:
                raise ValueError(f"cos and sin must be contiguous float32 [max_pos, r / 2] on the pool's device, "
                                 f"2 <= r <= {d}")
    r = _lib.Kv4Rows(q_ptr, k_ptr, v_ptr, o_ptr, q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head,
                     _ints(pos, "pos", dev, n), None if seq is None else _ints(seq, "seq", dev, n),
                     None if cos is None else cos.data_ptr(), None if sin is None else sin.data_ptr(), dtype, o_type, n,
                     heads, rotary, 1 if interleaved else 0, max_pos)
    if n:
        _lib.check(_lib.load().b2d_kv4_append(ctypes.byref(c), ctypes.byref(r), _stream_on(stream, dev)),
                   "b2d_kv4_append")
    return q_out


def kv4_read(pool, pos, table, *, seq=None, dtype=torch.bfloat16, status=None, stream=None):
    """The rows at positions ``pos`` of the sequences ``seq`` (as in
    ``kv4_append``) as values: ``(k, v)``, each [n, n_kv, d] of ``dtype``
    (float32, bf16 or fp16, all exact); zeros where ``pos`` is negative."""
    c, dev, _, table_rows, n_kv, d = _cache(pool, table, status)
    n = pos.numel()
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, bfloat16 or float16")
    if seq is None and n > table_rows:
        raise ValueError("more rows than table rows need seq")
    p, s = _ints(pos, "pos", dev, n), None if seq is None else _ints(seq, "seq", dev, n)
    if stream is None:
        k = pool.new_empty((n, n_kv, d), dtype=dtype)
    else:
        with torch.cuda.stream(stream):
            k = pool.new_empty((n, n_kv, d), dtype=dtype)
    v = _empty_like(k, stream)
    if n:
        _lib.check(_lib.load().b2d_kv4_read(ctypes.byref(c), p, s, n, _TYPES[dtype], k.data_ptr(), v.data_ptr(),
                                            _stream_on(stream, dev)), "b2d_kv4_read")
    return k, v


_QUERY_TYPES = (torch.bfloat16, torch.float16)


def kv4_attention(q, pool, lens, table, *, q_start=None, max_rows=None, max_len=None, scale=None, out=None,
                  status=None, stream=None):
    """Causal attention of the rows ``q`` [n, heads, d] (bf16 or fp16) over the
    4-bit cache; returns ``out`` (default: a new tensor of q's shape and type;
    may be ``q``).

    Sequence i (row i of ``table``) has ``lens[i]`` positions in the cache
    (int32; 0: its rows see nothing and become 0).  Decode: one row a
    sequence.  With ``q_start`` (int32 [n_seqs + 1]) sequence i has the rows
    q_start[i] .. q_start[i + 1], its last positions; none has more than
    ``max_rows`` (default: n), and rows of no sequence stay as they are.
    ``max_len`` (default: what a table row holds) bounds ``lens``; a close
    bound splits long sequences better.  ``scale`` defaults to d ** -0.5."""
    c, dev, bps, table_rows, n_kv, d = _cache(pool, table, status)
    n, heads = q.shape[:2] if q.dim() == 3 else (0, 0)
    shape = (n, heads, d)
    q_ptr, q_row, q_head = _strides(q, "q", dev, shape, _QUERY_TYPES)
    if heads < 1 or heads % n_kv:
        raise ValueError(f"q must have a multiple of {n_kv} heads")
    n_seqs = lens.numel()
    if n_seqs > table_rows:
        raise ValueError("more lengths than table rows")
    given = out is not None
    if not given:
        out = _empty_like(q, stream)
    o_ptr, o_row, o_head = _strides(out, "out", dev, shape, (q.dtype,))
    if given and (_folded(out) or (not _same_place(out, q) and _overlap(out, q))):
        raise ValueError("out must be q or apart from it")
    room = min(bps * PAGE_TOKENS, 2 ** 31 - 1)
    max_len = room if max_len is None else int(max_len)
    if not 0 <= max_len <= room:
        raise ValueError(f"max_len must be in [0, {room}] (the table's rows)")
    lens_ptr, start_ptr = _ints(lens, "lens", dev, n_seqs), None
    if q_start is None:
        if n_seqs != n or max_rows not in (None, 1):
            raise ValueError("without q_start there is one row a sequence")
        max_rows = 1
    else:
        start_ptr = _ints(q_start, "q_start", dev, n_seqs + 1)
        max_rows = max(1, n) if max_rows is None else int(max_rows)
        if max_rows < 1:
            raise ValueError("max_rows must be at least 1")
        max_rows = min(max_rows, max(1, n))
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale must be positive")
    if not n or not n_seqs:
        return out
    need, scratch_ptr = _scratch_bytes(dev, n_kv, d, heads, n_seqs, max_rows, max_len), None
    if need:  # from the stream's own memory: calls on other streams, and other graphs, have theirs
        if stream is None:
            scratch = pool.new_empty(need)
        else:
            with torch.cuda.stream(stream):
                scratch = pool.new_empty(need)
        scratch_ptr = scratch.data_ptr()
    query = _lib.Kv4Query(q_ptr, o_ptr, q_row, q_head, o_row, o_head, lens_ptr, start_ptr, _TYPES[q.dtype], n, heads,
                          n_seqs, max_rows, max_len, scale)
    _lib.check(_lib.load().b2d_kv4_attention(ctypes.byref(c), ctypes.byref(query), scratch_ptr, need,
                                             _stream_on(stream, dev)), "b2d_kv4_attention")
    return out
