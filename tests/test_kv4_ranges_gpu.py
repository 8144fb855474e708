"""GPU: the 4-bit cache's operators at the ends of their ranges, against their
definition in 64 bits (tests/kv4_ref.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_ref as R
from transformer_b200.kv4 import check_status, kv4_append, kv4_attention, kv4_read, new_kv4_pool

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def f64(t):
    return t.double().cpu().numpy()


def i32(a, dev):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32).to(dev)


def filled(k, v, cuda):
    """A cache of one sequence that holds the rows k, v [length, n_kv, d]:
    (pool, table, the held rows in 64 bits)."""
    length, n_kv, d = k.shape
    pages = (length + 15) // 16
    pool = new_kv4_pool(pages, n_kv, d, cuda)
    table = i32(np.random.default_rng(length).permutation(pages)[None], cuda)
    at, zero = i32(np.arange(length), cuda), i32(np.zeros(length), cuda)
    kv4_append(pool, *(torch.from_numpy(x.astype(np.float32)).to(cuda) for x in (k, v)), at, table, seq=zero)
    return pool, table, *(f64(x) for x in kv4_read(pool, at, table, seq=zero, dtype=torch.float32))


# a length, the rows that ask, heads a kv head: one token alone, with two blocks of
# columns, and split over the positions; a prompt's chunk of one group of columns
# and split over the positions
SHAPES = [(50, 1, 4), (50, 3, 5), (4001, 1, 4), (130, 40, 2), (4100, 35, 3)]


@pytest.mark.parametrize("length,rows,group", SHAPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("apart", [20, 27, 34])
def test_queries_of_wide_range(cuda, length, rows, group, d, apart):
    """bf16 query dims 2^apart below the row's largest count like the others:
    the keys are as much larger there, so both halves of the dims make the score."""
    rng = np.random.default_rng(length + d + apart)
    n_kv, far = 2, 2.0 ** (apart / 2)
    ratio = np.where(np.arange(d) % 32 < 16, far, 1 / far)  # (scales are per 16 dims)
    k = rng.normal(size=(length, n_kv, d)) / ratio * np.minimum(1, 2000 / far)  # (held magnitudes reach 64512)
    pool, table, hk, hv = filled(k, rng.normal(size=k.shape), cuda)
    q = torch.from_numpy(rng.normal(size=(rows, n_kv * group, d)) * ratio * np.maximum(1, far / 2000))
    q = q.to(torch.bfloat16).to(cuda)
    start = None if rows == 1 else i32([0, rows], cuda)
    out = kv4_attention(q, pool, i32([length], cuda), table, q_start=start)
    want, mass, size = R.attention(f64(q), hk, hv, d ** -0.5)
    bound = R.attention_bound(want, mass, size, length, d, 2.0 ** -8, np.abs(hv).max())
    err = np.abs(f64(out) - want)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("length,rows,group", SHAPES)
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("f16", 64), ("bf16", 128), ("f16", 128)])
@pytest.mark.parametrize("top", [1.0, 2.0 ** 5, 2.0 ** 11])
def test_scores_of_any_size(cuda, length, rows, group, dtype, d, top):
    """Scores to 2^30: finite, and shares of the rows that reach the largest.
    Keys are 0 or the cache's largest value, queries small whole numbers times
    `top`, so that every score is exact in 32 bits: those that are not the
    row's largest are too far below it to count."""
    rng = np.random.default_rng(length + d + int(top))
    n_kv, held = 2, 64512.0
    k = held * rng.integers(-1, 2, size=(7, n_kv, d))[rng.integers(0, 7, length)]  # seven rows, each many times
    pool, table, hk, hv = filled(k, rng.normal(size=k.shape), cuda)
    assert np.array_equal(hk, k)
    q = top * rng.integers(-15, 16, size=(rows, n_kv * group, d))
    out = kv4_attention(torch.from_numpy(q).to(TYPES[dtype]).to(cuda), pool, i32([length], cuda), table,
                        q_start=None if rows == 1 else i32([0, rows], cuda))
    want, mass, _ = R.attention(q, hk, hv, d ** -0.5)
    # (no score is off, and none that counts has an argument other than 0)
    bound = R.attention_bound(want, mass, 0.0, length, d, torch.finfo(TYPES[dtype]).eps / 2, np.abs(hv).max())
    err = np.abs(f64(out) - want)
    assert (err <= bound).all(), float(np.nanmax(err / bound))


@pytest.mark.parametrize("dtype,heads,n_kv,d,lens,rows", [
    ("bf16", 16, 4, 64, [1, 17, 64, 130, 333, 48], None), ("f16", 10, 2, 128, [70, 16, 5000], None),
    ("bf16", 8, 8, 128, [9001], None), ("bf16", 8, 2, 64, [130, 77], [40, 77]), ("f16", 32, 8, 128, [260, 70], [90, 70]),
    ("f16", 8, 2, 128, [5003, 4100], [70, 33]), ("bf16", 16, 4, 64, [700, 400, 720], [600, 350, 600])])
def test_blocks_that_the_table_does_not_name(cuda, dtype, heads, n_kv, d, lens, rows):
    """A row that sees a position of one is zero, others (before it) as ever, and
    the status is set.  One token alone, split, with two blocks of columns; chunks
    of one and two groups of columns, and split."""
    rng = np.random.default_rng(sum(lens) + d)
    bps, counts = (max(lens) + 15) // 16, rows or [1] * len(lens)
    blocks = len(lens) * bps
    pool, table = new_kv4_pool(blocks, n_kv, d, cuda), rng.permutation(blocks).reshape(len(lens), bps)
    held = []
    for i, n in enumerate(lens):
        k, v = (torch.from_numpy(rng.normal(size=(n, n_kv, d)).astype(np.float32)).to(cuda) for _ in range(2))
        at, seq = i32(np.arange(n), cuda), i32(np.full(n, i), cuda)
        kv4_append(pool, k, v, at, i32(table, cuda), seq=seq)
        held.append([f64(x) for x in kv4_read(pool, at, i32(table, cuda), seq=seq, dtype=torch.float32)])
    lost = np.zeros(table.shape, bool)
    lost[0, (lens[0] - counts[0] // 2 - 1) // 16] = True  # seen by a token, by half of a chunk's rows
    lost[-1, rng.integers(0, (lens[-1] + 15) // 16, 2)] = True
    bad = np.where(lost, rng.choice([-1, blocks, 2 ** 31 - 1, -2 ** 31], table.shape), table)
    q = torch.from_numpy(rng.normal(size=(sum(counts), heads, d))).to(TYPES[dtype]).to(cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    start = None if rows is None else i32(np.cumsum([0, *rows]), cuda)
    out = kv4_attention(q, pool, i32(lens, cuda), i32(bad, cuda), q_start=start, status=status)
    assert int(status.item()) == 0x203
    at, some = 0, False
    for i, (n, c, (k, v)) in enumerate(zip(lens, counts, held)):
        want, mass, size = R.attention(f64(q)[at:at + c], k, v, d ** -0.5)
        bound = R.attention_bound(want, mass, size, n, d, torch.finfo(TYPES[dtype]).eps / 2, np.abs(v).max())
        first = np.flatnonzero(lost[i, :(n + 15) // 16])
        zero = np.arange(n - c, n) >= (16 * first[0] if first.size else n)
        want[zero], bound[zero] = 0.0, 0.0
        err = np.abs(f64(out)[at:at + c] - want)
        assert (err <= bound).all(), i
        some = some or (zero.any() and not zero.all())
        at += c
    assert some or rows is None  # (rows on both sides of a lost block)


@pytest.mark.parametrize("n", [7, 600])  # (a block per batch of heads, a warp a row)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_skips_a_row_past_the_table_with_its_query(cuda, n, dtype):
    """A position past the table's row, a block that the pool does not have and a
    row that the table does not have: neither the pool nor q_out is written, in
    place either; the other rows are as without them."""
    t = TYPES.get(dtype, torch.float32)
    heads, n_kv, d, bps = 5, 2, 64, 3
    gen = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(n, h, d, generator=gen).to(t).to(cuda) for h in (heads, n_kv, n_kv))
    ang = torch.randn(200, d // 2, generator=gen)
    kw = dict(cos=ang.cos().to(cuda), sin=ang.sin().to(cuda))
    table = np.arange(n * bps).reshape(n, bps)
    pos, seq = np.arange(n) % 48, np.arange(n)
    bad = np.array([1, 3, 4, n - 1])
    pos[1], seq[4] = 16 * bps + 5, n
    table[3, pos[3] // 16], table[n - 1, pos[n - 1] // 16] = n * bps, -1
    good = torch.ones(n, dtype=torch.bool, device=cuda)
    good[torch.from_numpy(bad).to(cuda)] = False
    want_pool, pool = (new_kv4_pool(n * bps, n_kv, d, cuda) for _ in range(2))
    at, rows, table = i32(pos, cuda), i32(seq, cuda), i32(table, cuda)
    want = kv4_append(want_pool, k[good], v[good], at[good], table, seq=rows[good], q=q[good], **kw)
    for inplace in (False, True):
        pool.zero_()
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        src = q.clone()
        out = src if inplace else torch.full_like(q, 9.0)
        kv4_append(pool, k, v, at, table, seq=rows, q=src, q_out=out, status=status, **kw)
        assert int(status.item()) == 0x203 and torch.equal(pool, want_pool) and torch.equal(out[good], want)
        assert torch.equal(out[~good], q[~good] if inplace else torch.full_like(q[~good], 9.0))


@pytest.mark.parametrize("dtype,heads,n_kv,d,lens,rows", [
    ("bf16", 16, 4, 64, [1, 17, 333, 0], None), ("f16", 10, 2, 128, [70, 5000], None),
    ("f16", 8, 2, 128, [130, 77], [100, 77]), ("bf16", 8, 2, 64, [4097], [70])])
def test_attention_onto_its_queries(cuda, dtype, heads, n_kv, d, lens, rows):
    """out = q, contiguous and as a part of packed rows: what a separate out has."""
    t, counts = TYPES[dtype], rows or [1] * len(lens)
    n, bps = sum(counts), (max(lens) + 15) // 16
    gen = torch.Generator().manual_seed(n + d)
    pool, table = new_kv4_pool(len(lens) * bps, n_kv, d, cuda), i32(np.arange(len(lens) * bps).reshape(len(lens), bps), cuda)
    for i, length in enumerate(lens):
        k = torch.randn(length, n_kv, d, generator=gen).to(cuda)
        kv4_append(pool, k, k, i32(np.arange(length), cuda), table, seq=i32(np.full(length, i), cuda))
    packed = torch.randn(n, heads + 2 * n_kv, d, generator=gen).to(t).to(cuda)
    q, rest = packed[:, :heads], packed[:, heads:].clone()
    kw = dict(q_start=None if rows is None else i32(np.cumsum([0, *rows]), cuda))
    want = kv4_attention(q, pool, i32(lens, cuda), table, **kw)
    alone = q.contiguous()
    for x in (alone, q):
        assert kv4_attention(x, pool, i32(lens, cuda), table, out=x, **kw) is x and torch.equal(x, want)
    assert torch.equal(packed[:, heads:], rest)


def test_outputs_that_overlap_inputs_in_part_are_refused(cuda):
    from transformer_b200.generate import adjust_logits
    n, d = 4, 64
    buf = torch.zeros(n + 1, 9, d, device=cuda)
    q, k, v = buf[:n, :4], buf[:n, 4:6], buf[:n, 6:8]
    pool, table, pos = new_kv4_pool(n, 2, d, cuda), i32(np.arange(n)[:, None], cuda), i32(np.zeros(n), cuda)
    for out in (buf[1:, :4], buf[:n, 1:5], buf[:n, 4:8], buf.view(-1)[1:].as_strided((n, 4, d), q.stride()),
                buf.view(-1).as_strided((n, 4, d), (5 * d, d, 1)), torch.zeros(n, 1, d, device=cuda).expand(n, 4, d),
                buf.view(torch.bfloat16)[:n, :4, :d]):
        with pytest.raises(ValueError):
            kv4_append(pool, k, v, pos, table, q=q, q_out=out)
    assert torch.count_nonzero(pool) == 0 and torch.count_nonzero(buf) == 0
    for out in (q, torch.empty(n, 4, d, dtype=torch.float16, device=cuda)):
        assert kv4_append(pool, k, v, pos, table, q=q, q_out=out) is out
    h = torch.zeros(n + 1, 9, d, device=cuda, dtype=torch.bfloat16)
    lens = i32(np.ones(n), cuda)
    for out in (h[1:, :4], h[:n, 1:5], h.view(-1)[1:].as_strided((n, 4, d), h.stride()),
                torch.zeros(1, 4, d, device=cuda, dtype=torch.bfloat16).expand(n, 4, d)):
        with pytest.raises(ValueError):
            kv4_attention(h[:n, :4], pool, lens, table, out=out)
    kv4_attention(h[:n, :4], pool, lens, table, out=h[:n, 4:8])
    flat = torch.zeros(300, device=cuda)
    lg = flat.as_strided((3, 50), (100, 1))
    for out in (flat[1:].as_strided((3, 50), (100, 1)), flat[100:].as_strided((2, 50), (100, 1)),
                flat.as_strided((3, 50), (50, 1)), flat[49:].as_strided((3, 50), (100, 1))):
        with pytest.raises(ValueError):
            adjust_logits(lg[:out.shape[0]], out=out)
    other = flat[50:].as_strided((3, 50), (100, 1))  # the other half of each row
    assert adjust_logits(lg, out=other) is other and adjust_logits(lg, out=lg) is lg


@pytest.mark.parametrize("dtype,heads,n_kv,d", [("bf16", 16, 4, 64), ("f16", 12, 6, 128)])
def test_attention_of_many_short_chunks(cuda, dtype, heads, n_kv, d):
    """More sequences and kv heads than SMs, each with one tile of 128 columns,
    some with few rows, none, or more than positions."""
    rng = np.random.default_rng(d)
    n_seqs, bps, top = 45, 9, 128 // (heads // n_kv)
    rows = rng.integers(0, top + 1, n_seqs)
    lens = np.minimum(rows + rng.integers(-3, 90, n_seqs).clip(-3), 16 * bps).clip(0)
    rows[:3], lens[:3] = (top, 0, top), (16 * bps, 20, 0)
    pool, table = new_kv4_pool(n_seqs * bps, n_kv, d, cuda), i32(rng.permutation(n_seqs * bps).reshape(n_seqs, bps), cuda)
    at, seq = i32(np.concatenate([np.arange(x) for x in lens]), cuda), i32(np.repeat(np.arange(n_seqs), lens), cuda)
    k, v = (torch.from_numpy(rng.normal(size=(int(lens.sum()), n_kv, d)).astype(np.float32)).to(cuda) for _ in range(2))
    kv4_append(pool, k, v, at, table, seq=seq)
    held = [f64(x) for x in kv4_read(pool, at, table, seq=seq, dtype=torch.float32)]
    q = torch.from_numpy(rng.normal(size=(int(rows.sum()), heads, d))).to(TYPES[dtype]).to(cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = kv4_attention(q, pool, i32(lens, cuda), table, q_start=i32(np.cumsum([0, *rows]), cuda), max_rows=top,
                        status=status)
    check_status(status)
    a = b = 0
    for n, c in zip(lens, rows):
        hk, hv = (x[b:b + n] for x in held)
        want, mass, size = R.attention(f64(q)[a:a + c], hk, hv, d ** -0.5)
        bound = R.attention_bound(want, mass, size, max(n, 1), d, torch.finfo(TYPES[dtype]).eps / 2,
                                  np.abs(hv).max(initial=0))
        assert (np.abs(f64(out)[a:a + c] - want) <= bound).all()
        a, b = a + c, b + n


@pytest.mark.parametrize("n", [300, 512, 1024])  # (few rows, and a warp a row from 8 d on)
@pytest.mark.parametrize("q_type", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d,rotary", [(64, 64), (64, 32), (128, 128)])
def test_append_of_float32_rows(cuda, n, q_type, d, rotary):
    """What a model's pass of prompts appends: float32 rows of a packed
    projection, queries into another type, the halves of a head rotated."""
    heads, n_kv, t = 5, 2, TYPES.get(q_type, torch.float32)
    gen = torch.Generator().manual_seed(n + d + rotary)
    x = torch.randn(n, heads + 2 * n_kv, d, generator=gen).to(cuda)
    q, k, v = x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:]
    ang = torch.randn(n, rotary // 2, generator=gen)
    cos, sin = ang.cos().to(cuda), ang.sin().to(cuda)
    pages = (n + 15) // 16
    rng = np.random.default_rng(n)
    pool, table = new_kv4_pool(pages, n_kv, d, cuda), i32(rng.permutation(pages)[None], cuda)
    order = rng.permutation(n)
    pos, seq = i32(order, cuda), i32(np.zeros(n), cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.empty(n, heads, d, dtype=t, device=cuda)
    kv4_append(pool, k, v, pos, table, seq=seq, q=q, q_out=out, cos=cos, sin=sin, status=status)
    check_status(status)
    c, s = f64(cos)[order], f64(sin)[order]
    got_k, got_v = kv4_read(pool, pos, table, seq=seq, dtype=torch.float32)
    assert np.array_equal(f64(got_k), R.held(R.turned(f64(k), c, s, False)))
    assert np.array_equal(f64(got_v), R.held(f64(v)))
    # two products and a sum in float32 (3 2^-24 of |x| + |partner|), then one rounding
    # (an fp16 one is off by up to 2^-25 however small the number)
    want, pair = R.turned(f64(q), c, s, False), 2 * np.abs(f64(q)).max(-1, keepdims=True)
    work = 3 * 2.0 ** -24 * pair
    bound = torch.finfo(t).eps / 2 * (np.abs(want) + work) + work + (2.0 ** -25 if q_type == "f16" else 0.0)
    assert (np.abs(f64(out) - want) <= bound).all()
