"""The paged KV cache in 4 bits: append, read-back and attention as operators.

``DecodeEngine(w, max_batch, kv_bits=4)`` decodes and serves from such a cache;
the functions here are its parts, for one layer's pool of any ``n_kv`` heads of
64 or 128 dims (``b2d_kv4_*`` in include/b2d.h, which states the format: groups
of 16 dims with a scale of 8 bits, 4.5 bits a value, and held values exact in
bf16 and fp16).  The reference has no cache below bf16.

All calls are asynchronous and stream-ordered.  A pool is the uint8 tensor of
``new_kv4_pool``; a block of it holds 16 positions; ``table`` int32
[n_seqs, blocks_per_seq] names the block of positions 16i.. of each sequence.
Entries are read only where a position needs them.  Bad entries, positions and
lengths seen by a kernel set ``status`` (an int32 tensor of one item, 0 at
first) and skip the access; ``check_status`` raises for it.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

PAGE_TOKENS = 16  # positions per block
_TYPES = {torch.float32: _lib.B2D_F32, torch.bfloat16: _lib.B2D_BF16, torch.float16: _lib.B2D_F16}


def _stream_on(stream, device) -> ctypes.c_void_p:
    """The stream's handle, by default the current one of ``device``."""
    return ctypes.c_void_p((stream or torch.cuda.current_stream(device)).cuda_stream)


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


def _ints(t, name, device, n):
    if t.dtype != torch.int32 or t.device != device or t.dim() != 1 or not t.is_contiguous() or t.numel() != n:
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} items on {device}")
    return t.data_ptr()


def _cache(pool, table, status, n_kv, d) -> _lib.Kv4Cache:
    if pool.device.type != "cuda":
        raise ValueError("pool must be on a GPU")
    if pool.dtype != torch.uint8 or pool.dim() != 3 or not pool.is_contiguous() or tuple(pool.shape[1:]) != (
            n_kv, page_bytes(d)) or pool.shape[0] < 1:
        raise ValueError(f"pool must be contiguous uint8 [num_blocks, {n_kv}, {page_bytes(d)}] (see new_kv4_pool)")
    if table.dtype != torch.int32 or table.device != pool.device or table.dim() != 2 or not table.is_contiguous() or (
            table.numel() < 1):
        raise ValueError("table must be a contiguous int32 [n_seqs, blocks_per_seq] tensor on the pool's device")
    if status is not None and (status.dtype != torch.int32 or status.device != pool.device or status.numel() != 1):
        raise ValueError("status must be an int32 tensor of one item on the pool's device")
    return _lib.Kv4Cache(pool.data_ptr(), table.data_ptr(), status.data_ptr() if status is not None else None, n_kv, d,
                         pool.shape[0], table.shape[1], table.shape[0], pool.device.index or 0)


def _heads(t, name, device, dtype=None, rows=None):
    """[rows, heads, d] with contiguous dims; any row and head strides."""
    if t.dim() != 3 or t.device != device or t.dtype not in _TYPES or (dtype is not None and t.dtype != dtype) or (
            rows is not None and t.shape[0] != rows) or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name} must be a [rows, heads, d] tensor on {device} with contiguous dims"
                         + (f" of type {dtype}" if dtype is not None else ""))
    return t.data_ptr()


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
    returned.  Two rows at one position: the cache gets dims of either."""
    d = k.shape[-1] if k.dim() == 3 else 0
    c = _cache(pool, table, status, k.shape[1] if k.dim() == 3 else 0, d)
    dev, n = pool.device, k.shape[0]
    r = _lib.Kv4Rows(k=_heads(k, "k", dev), v=_heads(v, "v", dev, k.dtype, n), dtype=_TYPES[k.dtype], n_rows=n,
                     k_row=k.stride(0), k_head=k.stride(1), v_row=v.stride(0), v_head=v.stride(1))
    if v.shape != k.shape:
        raise ValueError("v must have k's shape")
    r.pos = _ints(pos, "pos", dev, n)
    if seq is not None:
        r.seq = _ints(seq, "seq", dev, n)
    elif n > table.shape[0]:
        raise ValueError("more rows than table rows need seq")
    if q is not None:
        r.q = _heads(q, "q", dev, k.dtype, n)
        if q.shape[2] != d or q.shape[1] < 1:
            raise ValueError("q must have heads of k's dims")
        if q_out is None:
            with torch.cuda.stream(stream or torch.cuda.current_stream(dev)):
                q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        r.q_out = _heads(q_out, "q_out", dev, None if q.dtype == torch.float32 else q.dtype, n)
        if q_out.shape != q.shape or (q_out.data_ptr() == q.data_ptr() and
                                      (q_out.stride() != q.stride() or q_out.dtype != q.dtype)):
            raise ValueError("q_out must have q's shape (and be q or apart from it)")
        r.q_row, r.q_head, r.q_out_row, r.q_out_head = q.stride(0), q.stride(1), q_out.stride(0), q_out.stride(1)
        r.n_heads, r.q_out_dtype = q.shape[1], _TYPES[q_out.dtype]
    elif q_out is not None:
        raise ValueError("q_out without q")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        for t, name in ((cos, "cos"), (sin, "sin")):
            if t.dtype != torch.float32 or t.device != dev or t.dim() != 2 or not t.is_contiguous() or (
                    t.shape != cos.shape) or not 1 <= 2 * t.shape[1] <= d or t.shape[0] < 1:
                raise ValueError(f"{name} must be contiguous float32 [max_pos, r / 2] with 2 <= r <= {d} on {dev}")
        r.cos, r.sin, r.rotary_dim, r.max_pos = cos.data_ptr(), sin.data_ptr(), 2 * cos.shape[1], cos.shape[0]
        r.interleaved = int(bool(interleaved))
    if n:
        _lib.check(_lib.load().b2d_kv4_append(ctypes.byref(c), ctypes.byref(r), _stream_on(stream, dev)),
                   "b2d_kv4_append")
    return q_out


def kv4_read(pool, pos, table, *, seq=None, dtype=torch.bfloat16, status=None, stream=None):
    """The rows at positions ``pos`` of the sequences ``seq`` (as in
    ``kv4_append``) as values: ``(k, v)``, each [n, n_kv, d] of ``dtype``
    (float32, bf16 or fp16, all exact); zeros where ``pos`` is negative."""
    n_kv, d = (pool.shape[1], pool.shape[2] // 18) if pool.dim() == 3 else (0, 0)
    c = _cache(pool, table, status, n_kv, d)
    dev, n = pool.device, pos.numel()
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, bfloat16 or float16")
    if seq is None and n > table.shape[0]:
        raise ValueError("more rows than table rows need seq")
    p, s = _ints(pos, "pos", dev, n), _ints(seq, "seq", dev, n) if seq is not None else None
    with torch.cuda.stream(stream or torch.cuda.current_stream(dev)):
        k, v = (torch.empty(n, n_kv, d, dtype=dtype, device=dev) for _ in range(2))
    if n:
        _lib.check(_lib.load().b2d_kv4_read(ctypes.byref(c), p, s, n, _TYPES[dtype], k.data_ptr(), v.data_ptr(),
                                            _stream_on(stream, dev)), "b2d_kv4_read")
    return k, v


def kv4_attention(q, pool, lens, table, *, q_start=None, max_rows=None, max_len=None, scale=None, out=None,
                  status=None, stream=None):
    """Causal attention of the rows ``q`` [n, heads, d] (bf16 or fp16) over the
    4-bit cache; returns ``out`` (default: a new tensor of q's shape and type).

    Sequence i (row i of ``table``) has ``lens[i]`` positions in the cache
    (int32; 0: its rows see nothing and become 0).  Decode: one row a
    sequence.  With ``q_start`` (int32 [n_seqs + 1]) sequence i has the rows
    q_start[i] .. q_start[i + 1], its last positions; none has more than
    ``max_rows`` (default: n), and rows of no sequence stay as they are.
    ``max_len`` (default: what a table row holds) bounds ``lens``; a close
    bound splits long sequences better.  ``scale`` defaults to d ** -0.5."""
    n_kv, d = (pool.shape[1], pool.shape[2] // 18) if pool.dim() == 3 else (0, 0)
    c = _cache(pool, table, status, n_kv, d)
    dev = pool.device
    _heads(q, "q", dev)
    n, heads = q.shape[:2]
    if q.dtype not in (torch.bfloat16, torch.float16) or q.shape[2] != d or heads < 1 or heads % n_kv:
        raise ValueError(f"q must be bf16 or fp16 [rows, a multiple of {n_kv} heads, {d}]")
    n_seqs = lens.numel()
    if n_seqs > table.shape[0]:
        raise ValueError("more lengths than table rows")
    if q_start is None and n_seqs != n:
        raise ValueError("without q_start there is one row a sequence")
    if out is None:
        with torch.cuda.stream(stream or torch.cuda.current_stream(dev)):
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    _heads(out, "out", dev, q.dtype, n)
    if out.shape != q.shape:
        raise ValueError("out must have q's shape")
    room = min(table.shape[1] * PAGE_TOKENS, 2 ** 31 - 1)
    max_len = room if max_len is None else int(max_len)
    max_rows = (1 if q_start is None else max(1, n)) if max_rows is None else int(max_rows)
    if not 0 <= max_len <= room:
        raise ValueError(f"max_len must be in [0, {room}] (the table's rows)")
    if max_rows < 1 or (q_start is None and max_rows != 1):
        raise ValueError("max_rows must be at least 1, and 1 without q_start")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale must be positive")
    query = _lib.Kv4Query(q.data_ptr(), out.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                          _ints(lens, "lens", dev, n_seqs),
                          _ints(q_start, "q_start", dev, n_seqs + 1) if q_start is not None else None,
                          _TYPES[q.dtype], n, heads, n_seqs, max_rows, max_len, scale)
    if not n or not n_seqs:
        return out
    lib, need = _lib.load(), ctypes.c_uint64()
    _lib.check(lib.b2d_kv4_attention_scratch(ctypes.byref(c), ctypes.byref(query), ctypes.byref(need)),
               "b2d_kv4_attention_scratch")
    scratch = None
    if need.value:  # from the stream's own memory: calls on other streams, and other graphs, have theirs
        with torch.cuda.stream(stream or torch.cuda.current_stream(dev)):
            scratch = torch.empty(need.value, dtype=torch.uint8, device=dev)
    _lib.check(lib.b2d_kv4_attention(ctypes.byref(c), ctypes.byref(query),
                                     scratch.data_ptr() if scratch is not None else None, need.value,
                                     _stream_on(stream, dev)), "b2d_kv4_attention")
    return out
