"""GPU: the 4-bit paged KV cache (append, read, attention) against its
definition in 64 bits (tests/kv4_ref.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_ref as R
from transformer_b200 import _lib
from transformer_b200.kv4 import check_status, kv4_append, kv4_attention, kv4_read, new_kv4_pool

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def f64(t):
    return t.double().cpu().numpy()


def i32(a, dev):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32).to(dev)


def angles(max_pos, r, dev):
    a = np.arange(max_pos)[:, None] * 10000.0 ** (-np.arange(0, r, 2) / r)
    return tuple(torch.from_numpy(f(a).astype(np.float32)).to(dev) for f in (np.cos, np.sin))


def random_pool(rng, blocks, n_kv, d, dev):
    """A pool of finite held values (every byte a legal one), as numpy and on the device."""
    pool = rng.integers(0, 256, (blocks, n_kv, 18 * d)).astype(np.uint8)
    for lo in (0, 9 * d):
        codes = pool[:, :, lo:lo + 8 * d]
        codes[(codes & 15) == 0] += 1    # code 0 (-8) is never written
        codes[codes < 16] += 16
        pool[:, :, lo + 8 * d:lo + 9 * d] = rng.integers(95, 108, (blocks, n_kv, d))  # scales 0.05 .. 0.18
    return pool, torch.from_numpy(pool).to(dev)


# ---- append and read ---------------------------------------------------------

@pytest.mark.parametrize("dtype,heads,n_kv,d,rope,rotary", [
    ("bf16", 16, 4, 64, "half", 64), ("f16", 8, 8, 128, "interleaved", 128), ("f32", 4, 2, 64, "half", 64),
    ("bf16", 5, 1, 128, "half", 96), ("f16", 6, 3, 64, "half", 2), ("f32", 3, 3, 128, "interleaved", 48),
    ("bf16", 10, 5, 64, "half", 36), ("bf16", 2, 2, 128, "none", 0)])
def test_append_holds_the_quantised_rotation(cuda, dtype, heads, n_kv, d, rope, rotary):
    """Every code and scale is the definition's for the exact rotation (held
    values compare equal), through packed rows, ragged sequences in any order
    and pages that end inside a sequence's rows."""
    rng = np.random.default_rng(heads * 1000 + d + rotary)
    t = TYPES[dtype]
    lens, rows = [37, 1, 16, 130], [37, 1, 5, 23]
    bps = 9
    table = rng.permutation(40)[:4 * bps].reshape(4, bps)
    seq = np.repeat(np.arange(4), rows)
    pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)])
    order = rng.permutation(pos.size)
    seq, pos = seq[order], pos[order]
    n = pos.size
    gen = torch.Generator().manual_seed(n + d)
    qkv = (torch.randn(n, (heads + 2 * n_kv) * d, generator=gen) *
           torch.exp(2 * torch.randn((heads + 2 * n_kv) * d, generator=gen))).to(t).to(cuda)
    q = qkv[:, :heads * d].view(n, heads, d)
    k = qkv[:, heads * d:(heads + n_kv) * d].view(n, n_kv, d)
    v = qkv[:, (heads + n_kv) * d:].view(n, n_kv, d)
    pool, status = new_kv4_pool(40, n_kv, d, cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    cos, sin = angles(144, rotary, cuda) if rotary else (None, None)
    seq_d, pos_d, table_d = i32(seq, cuda), i32(pos, cuda), i32(table, cuda)
    q_out = kv4_append(pool, k, v, pos_d, table_d, seq=seq_d, q=q, cos=cos, sin=sin,
                       interleaved=rope == "interleaved", status=status)
    check_status(status)
    want_q, want_k = f64(q), f64(k)
    if rotary:
        c, s = f64(cos)[pos], f64(sin)[pos]
        want_q, want_k = (R.turned(x, c, s, rope == "interleaved") for x in (want_q, want_k))
    for out in TYPES.values():
        got_k, got_v = kv4_read(pool, pos_d, table_d, seq=seq_d, dtype=out, status=status)
        assert np.array_equal(f64(got_k), R.held(want_k)) and np.array_equal(f64(got_v), R.held(f64(v)))
    # two products and a sum in float32, then one rounding: at most 3 2^-24 of
    # |x| + |partner| (each at most the pair's root of squares), and half a step
    pair = np.abs(f64(q)).max(-1, keepdims=True) * 2
    err = np.abs(f64(q_out) - want_q)
    assert (err <= torch.finfo(t).eps / 2 * (np.abs(want_q) + 3 * 2.0 ** -24 * pair) + 3 * 2.0 ** -24 * pair).all()
    # the layout: the same values by the documented bytes
    pages = R.page_values(pool.cpu().numpy(), d)
    at = table[seq, pos // 16]
    assert np.array_equal(pages[0][at, :, pos % 16], R.held(want_k))
    assert np.array_equal(pages[1][at, :, pos % 16], R.held(f64(v)))
    check_status(status)


def test_append_borders(cuda):
    """Values on the borders: amax an exact multiple of 7 (the scale must not
    step up), quotients at half (to even), tiny and huge groups, infinities
    and NaN."""
    rows = []
    for s in (2.0 ** -17, 5 * 2.0 ** -17, 2.0 ** -14, 1.125 * 2.0 ** -3, 1.875, 9216.0):
        g = np.array([7, -7, 0.5, 1.5, 2.5, -0.5, -1.5, -6.5, 6.5, 3.5, -4.5, 0, 1, 0.25, -0.75, 5.5]) * s
        rows.append(g)
        rows.append(np.where(np.abs(g) == 7 * s, g * (1 + 2.0 ** -7), g))  # just over: the next scale
    rows.append(np.zeros(16))
    rows.append(np.full(16, -0.0))
    rows.append(np.r_[np.full(8, 2.0 ** -130), np.full(8, -2.0 ** -126)])
    rows.append(np.r_[1e5, -3e38, np.zeros(12), 64512, -100])
    rows.append(np.r_[np.inf, -np.inf, np.zeros(12), 1e4, -9300])
    rows.append(np.r_[np.nan, 3.0, np.zeros(13), np.nan])
    rows.append(np.full(16, np.nan))
    while len(rows) % 4:
        rows.append(np.linspace(-1, 1, 16))
    x = torch.tensor(np.array(rows).reshape(-1, 1, 64), dtype=torch.float32).to(cuda)
    n = x.shape[0]
    pool = new_kv4_pool(1, 1, 64, cuda)
    pos, table = i32(np.arange(n), cuda), i32([[0]], cuda)
    zero = i32(np.zeros(n), cuda)
    kv4_append(pool, x, x, pos, table, seq=zero)
    k, v = kv4_read(pool, pos, table, seq=zero, dtype=torch.float32)
    want = R.held(f64(x))
    assert np.array_equal(f64(k), want) and np.array_equal(f64(v), want)


def test_append_decides_by_the_exact_rotation(cuda):
    """Keys whose rotated quotient lies within float32 rounding of a border:
    the code is the exact rotation's.  (Angles with many bits, 2^18 groups.)"""
    n, n_kv, d = 8192, 2, 64
    gen = torch.Generator().manual_seed(11)
    k = torch.randn(n, n_kv, d, generator=gen).to(cuda)
    cos, sin = angles(n, d, cuda)
    pool = new_kv4_pool(n // 16, n_kv, d, cuda)
    pos, table, zero = i32(np.arange(n), cuda), i32(np.arange(n // 16)[None], cuda), i32(np.zeros(n), cuda)
    kv4_append(pool, k, k, pos, table, seq=zero, cos=cos, sin=sin)
    got, _ = kv4_read(pool, pos, table, seq=zero, dtype=torch.float32)
    assert np.array_equal(f64(got), R.held(R.turned(f64(k), f64(cos), f64(sin), False)))


@pytest.mark.parametrize("d", [64, 128])
def test_append_touches_its_bytes_only(cuda, d):
    rng = np.random.default_rng(d)
    n_kv = 3
    before, pool = random_pool(rng, 6, n_kv, d, cuda)
    table = np.array([[4, 1], [2, 5]])
    seq, pos = np.array([0, 1, 1]), np.array([17, 3, 30])
    k = torch.from_numpy(rng.normal(size=(3, n_kv, d)).astype(np.float32)).to(cuda)
    kv4_append(pool, k, k, i32(pos, cuda), i32(table, cuda), seq=i32(seq, cuda))
    after = pool.cpu().numpy()
    mine = np.zeros_like(before, dtype=bool)
    for s, p in zip(seq, pos):
        for where in (R.k_bytes, R.v_bytes):
            for i in range(d):
                code, _, scale = where(d, p % 16, i)
                mine[table[s, p // 16], :, [code, scale]] = True
    assert np.array_equal(after[~mine], before[~mine])


def test_append_skips_idle_and_bad_rows(cuda):
    d, n_kv = 64, 2
    pool = new_kv4_pool(4, n_kv, d, cuda)
    cos, sin = angles(20, d, cuda)
    table = i32([[0, 1], [2, 9], [-1, 3]], cuda)
    k = torch.randn(1, n_kv, d, device=cuda)
    for seq, pos, word in ((0, -1, 0), (0, -2 ** 31, 0), (0, 20, 0x202), (1, 16, 0x203), (2, 3, 0x203), (3, 0, 0x203),
                           (-1, 0, 0x203)):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        q = torch.full((1, 2, d), 7.0, device=cuda)
        out = torch.full_like(q, -1.0)
        kv4_append(pool, k, k, i32([pos], cuda), table, seq=i32([seq], cuda), q=q, q_out=out, cos=cos, sin=sin,
                   status=status)
        assert int(status.item()) == word
        assert torch.count_nonzero(pool) == 0
        if word != 0x203:
            assert (out == -1).all()
        if word:
            with pytest.raises(_lib.B2DError):
                check_status(status)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    kv4_append(pool, k, k, i32([32], cuda), table, seq=i32([0], cuda), status=status)  # past the table row
    assert int(status.item()) == 0x203 and torch.count_nonzero(pool) == 0
    status.zero_()
    a, b = kv4_read(pool, i32([-1, 40, 3], cuda), table, seq=i32([0, 0, 2], cuda), status=status)
    assert torch.count_nonzero(a) == 0 and torch.count_nonzero(b) == 0 and int(status.item()) == 0x203


@pytest.mark.parametrize("dtype,heads,n_kv,d,rotary,interleaved", [
    ("bf16", 16, 4, 64, 64, False), ("f16", 7, 3, 128, 64, True), ("f32", 6, 2, 128, 100, False), ("bf16", 3, 3, 64, 0, False)])
def test_append_and_read_of_many_rows(cuda, dtype, heads, n_kv, d, rotary, interleaved):
    """A pass of many rows (another split of the work) holds and gives what small ones do."""
    n, t = 1100, TYPES[dtype]
    rng = np.random.default_rng(d + heads)
    gen = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn(n, h, d, generator=gen).to(t).to(cuda) for h in (heads, n_kv, n_kv))
    bps = (n + 15) // 16
    table = i32(rng.permutation(2 * bps)[:bps][None], cuda)
    pos, seq = i32(rng.permutation(n), cuda), i32([0] * n, cuda)
    ang = torch.randn(n, max(1, rotary // 2), generator=gen)
    kw = dict(cos=ang.cos().to(cuda), sin=ang.sin().to(cuda), interleaved=interleaved) if rotary else {}
    pools = [new_kv4_pool(2 * bps, n_kv, d, cuda) for _ in range(2)]
    whole = kv4_append(pools[0], k, v, pos, table, seq=seq, q=q, **kw)
    got = kv4_read(pools[0], pos, table, seq=seq, dtype=t)
    for lo in range(0, n, 300):
        c = slice(lo, min(n, lo + 300))
        part = kv4_append(pools[1], k[c], v[c], pos[c], table, seq=seq[c], q=q[c], **kw)
        assert torch.equal(part, whole[c])
    assert torch.equal(*pools)
    for lo in range(0, n, 300):
        c = slice(lo, min(n, lo + 300))
        for x, y in zip(got, kv4_read(pools[1], pos[c], table, seq=seq[c], dtype=t)):
            assert torch.equal(x[c], y)


def test_append_two_rows_at_one_position(cuda):
    """Bytes of both: finite, within the larger row's reach; other rows as alone."""
    rng = np.random.default_rng(41)
    n, n_kv, d = 6, 3, 128
    gen = torch.Generator().manual_seed(5)
    k = torch.randn(n, n_kv, d, generator=gen).to(cuda)
    v = 50 * torch.randn(n, n_kv, d, generator=gen).to(cuda)
    pos, table = i32([0, 7, 7, 7, 20, 3], cuda), i32(rng.permutation(4)[None, :2], cuda)
    seq = i32([0] * n, cuda)
    pool = new_kv4_pool(4, n_kv, d)
    kv4_append(pool, k, v, pos, table, seq=seq)
    got = kv4_read(pool, pos, table, seq=seq, dtype=torch.float32)
    for x, y in zip((k, v), got):
        assert torch.isfinite(y).all() and float(y[1:4].abs().max()) <= 1.15 * float(x[1:4].abs().max())
    keep = torch.tensor([0, 4, 5], device=cuda)
    alone = new_kv4_pool(4, n_kv, d)
    kv4_append(alone, k[keep], v[keep], pos[keep], table, seq=seq[:3])
    for y, z in zip(got, kv4_read(alone, pos[keep], table, seq=seq[:3], dtype=torch.float32)):
        assert torch.equal(y[keep], z)


def test_append_turns_q_in_place_and_unaligned_rows(cuda):
    """q_out = q gives what a separate q_out gives; rows that start off 16
    bytes (a view one element in) and strided heads give the same."""
    n, heads, n_kv, d = 9, 6, 2, 128
    gen = torch.Generator().manual_seed(2)
    base = torch.randn(n, heads + 2 * n_kv, d, generator=gen).to(torch.bfloat16).to(cuda)
    q, k, v = base[:, :heads], base[:, heads:heads + n_kv], base[:, heads + n_kv:]
    cos, sin = angles(64, d, cuda)
    pos, table = i32(np.arange(n) * 3, cuda), i32(np.arange(36).reshape(9, 4), cuda)

    def run(q, k, v, q_out=None):
        pool = new_kv4_pool(36, n_kv, d, cuda)
        return kv4_append(pool, k, v, pos, table, q=q, q_out=q_out, cos=cos, sin=sin), pool

    want, pool = run(q.contiguous(), k.contiguous(), v.contiguous())
    odd = torch.zeros(n, heads + 2 * n_kv, d + 3, dtype=torch.bfloat16, device=cuda)
    odd[:, :, 1:d + 1] = base
    odd = odd[:, :, 1:d + 1]
    out = torch.zeros(n, heads, d + 1, dtype=torch.bfloat16, device=cuda)[:, :, 1:]
    got, pool2 = run(odd[:, :heads], odd[:, heads:heads + n_kv], odd[:, heads + n_kv:], out)
    assert torch.equal(got, want) and torch.equal(pool2, pool)
    turned = base.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    got, pool3 = run(turned[:, :heads], turned[:, heads:heads + n_kv], turned[:, heads + n_kv:])
    assert torch.equal(got, want) and torch.equal(pool3, pool)
    got, pool4 = run(q, k, v, q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q, want) and torch.equal(pool4, pool)


def test_append_f32_rows_into_bf16_queries(cuda):
    n, d = 5, 64
    q = torch.randn(n, 4, d, device=cuda)
    k = torch.randn(n, 2, d, device=cuda)
    pool, table, pos = new_kv4_pool(n, 2, d, cuda), i32(np.arange(n)[:, None], cuda), i32(np.arange(n), cuda)
    cos, sin = angles(16, d, cuda)
    f = kv4_append(pool, k, k, pos, table, q=q, cos=cos, sin=sin)
    for t in (torch.bfloat16, torch.float16):
        o = kv4_append(pool, k, k, pos, table, q=q, q_out=torch.empty(n, 4, d, dtype=t, device=cuda), cos=cos, sin=sin)
        assert torch.equal(o, f.to(t))


# ---- attention -----------------------------------------------------------------

def check_attention(cuda, rng, dtype, heads, n_kv, d, lens, rows=None, max_len=None, trash=True, extra_rows=0,
                    scale=None, stream=None):
    """One call against the definition; slots past a sequence's end hold NaN scales."""
    t = TYPES[dtype]
    pages = [(n + 15) // 16 for n in lens]
    bps = max(1, max(pages)) + 1
    blocks = sum(pages) + 2
    pool_h, _ = random_pool(rng, blocks, n_kv, d, "cpu")
    perm = rng.permutation(blocks)
    table = np.full((len(lens), bps), -5)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = perm[at:at + p]
        at += p
    kp, vp = R.page_values(pool_h, d)
    if trash:
        for i, n in enumerate(lens):
            if n % 16:
                for r in range(n % 16, 16):
                    for where in (R.k_bytes, R.v_bytes):
                        for dim in range(0, d, 4):
                            pool_h[table[i, n // 16], :, where(d, r, dim)[2]] = 0xFF
    starts = None
    counts = [1] * len(lens) if rows is None else rows
    n_rows = sum(counts) + extra_rows
    gen = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
    q = torch.randn(n_rows, heads, d, generator=gen).to(t)
    if rows is not None:
        starts = i32(np.concatenate([[0], np.cumsum(rows)]), cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full((n_rows, heads, d), 3.0, dtype=t, device=cuda)
    args = (q.to(cuda), torch.from_numpy(pool_h).to(cuda), i32(lens, cuda), i32(table, cuda))
    torch.cuda.synchronize()
    kv4_attention(*args, q_start=starts, max_len=max_len, scale=scale, max_rows=max(rows) if rows else None, out=out,
                  status=status, stream=stream)
    torch.cuda.synchronize()
    check_status(status)
    got, at = f64(out), 0
    qn = f64(q)
    for i, (n, c) in enumerate(zip(lens, counts)):
        k, v = R.sequence(kp, table[i], n), R.sequence(vp, table[i], n)
        want, mass, size = R.attention(qn[at:at + c], k, v, d ** -0.5 if scale is None else scale)
        bound = R.attention_bound(want, mass, size, max(n, 1), d, torch.finfo(t).eps / 2, np.nanmax(np.abs(vp)))
        err = np.abs(got[at:at + c] - want)
        assert (err <= bound).all(), (i, n, c, float((err / bound).max()))
        at += c
    assert (got[at:] == 3.0).all()  # rows behind the last sequence
    return args, out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,n_kv,d", [(16, 4, 64), (8, 8, 64), (8, 1, 64), (32, 8, 128), (7, 7, 128), (10, 2, 128)])
def test_attention_one_row_a_sequence(cuda, dtype, heads, n_kv, d):
    rng = np.random.default_rng(heads * d)
    check_attention(cuda, rng, dtype, heads, n_kv, d, [1, 0, 15, 16, 17, 31, 64, 65, 200, 512, 2, 129])


@pytest.mark.parametrize("dtype,heads,n_kv,d", [("bf16", 16, 4, 64), ("f16", 32, 8, 128)])
def test_attention_one_long_sequence(cuda, dtype, heads, n_kv, d):
    """Split over the positions and joined; and the splits of a batch whose
    other rows have fewer of them, or none."""
    rng = np.random.default_rng(d)
    check_attention(cuda, rng, dtype, heads, n_kv, d, [9001])
    check_attention(cuda, rng, dtype, heads, n_kv, d, [3000, 0, 1, 129, 700])
    check_attention(cuda, rng, dtype, heads, n_kv, d, [40, 33], max_len=48)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 9, 16, 17, 32])
def test_attention_head_groups(cuda, group):
    rng = np.random.default_rng(group)
    check_attention(cuda, rng, "bf16", 2 * group, 2, 64, [70, 1, 300])
    check_attention(cuda, rng, "f16", group, 1, 128, [33, 16])


@pytest.mark.parametrize("dtype,heads,n_kv,d", [("bf16", 16, 4, 64), ("f16", 8, 2, 128), ("bf16", 3, 3, 128),
                                                ("f16", 12, 4, 64), ("bf16", 20, 1, 64)])
@pytest.mark.parametrize("lens,rows", [
    ([64], [64]), ([1], [1]), ([130, 40, 7], [130, 3, 7]), ([0, 20, 33], [2, 20, 0]), ([5, 300], [9, 77]),
    ([1025], [17]), ([260, 255, 16], [129, 128, 16])])
def test_attention_several_rows(cuda, dtype, heads, n_kv, d, lens, rows):
    """Chunks of prompts, causal: whole prompts, chunks on a longer past, an
    empty sequence with rows, one with no rows, more rows than positions (the
    first ones see nothing), and rows of no sequence."""
    rng = np.random.default_rng(sum(lens) + d)
    check_attention(cuda, rng, dtype, heads, n_kv, d, lens, rows, extra_rows=3)


@pytest.mark.parametrize("dtype,heads,n_kv,d", [("bf16", 16, 4, 64), ("f16", 8, 2, 128), ("bf16", 4, 4, 128)])
def test_attention_many_chunks(cuda, dtype, heads, n_kv, d):
    """More tiles of columns than SMs, so that a CTA takes two groups of them,
    the second one empty here and there: more sequences than are put in order of
    their lengths, and few of equal and unequal lengths."""
    rng = np.random.default_rng(heads + d)
    rows = [int(rng.integers(0, 161)) for _ in range(44)]
    check_attention(cuda, rng, dtype, heads, n_kv, d, [r + int(rng.integers(0, 60)) for r in rows], rows, extra_rows=2)
    rows = [600, 33, 350, 0, 600]
    check_attention(cuda, rng, dtype, heads, n_kv, d, [700, 90, 400, 90, 700], rows)


@pytest.mark.parametrize("dtype,heads,n_kv,d", [("bf16", 4, 4, 64), ("f16", 8, 2, 128)])
def test_attention_split_chunks(cuda, dtype, heads, n_kv, d):
    """Few columns on many positions, split and joined; one sequence has fewer splits."""
    rng = np.random.default_rng(heads)
    check_attention(cuda, rng, dtype, heads, n_kv, d, [5003, 1100, 70], [70, 66, 70])
    check_attention(cuda, rng, dtype, heads, n_kv, d, [4097], [150])


def test_attention_large_scores_and_scales(cuda):
    rng = np.random.default_rng(5)
    check_attention(cuda, rng, "bf16", 4, 2, 64, [100, 333], scale=3.0)
    check_attention(cuda, rng, "f16", 4, 2, 128, [100, 333], scale=1e-3)


def test_attention_extremes_of_the_cache(cuda):
    """The largest and smallest scales: 64512 in K and V, subnormal ones."""
    d = 64
    for t in ("bf16", "f16"):
        for mag in (64512.0, 2.0 ** -17 * 3):
            x = torch.zeros(20, 1, d, device=cuda)
            x[:, 0, ::3] = mag
            x[::2, 0, 5] = -mag
            pool, table = new_kv4_pool(2, 1, d, cuda), i32([[1, 0]], cuda)
            kv4_append(pool, x, x, i32(np.arange(20), cuda), table, seq=i32(np.zeros(20), cuda))
            q = torch.randn(1, 4, d, generator=torch.Generator().manual_seed(1)).to(TYPES[t]).to(cuda)
            scale = 1e-5 if mag > 1 else 0.125
            o = kv4_attention(q, pool, i32([20], cuda), table, scale=scale)
            k = R.held(f64(x))
            want, mass, size = R.attention(f64(q), k, k, scale)
            bound = R.attention_bound(want, mass, size, 20, d, torch.finfo(TYPES[t]).eps / 2, np.abs(k).max())
            assert (np.abs(f64(o) - want) <= bound).all()


def test_attention_bad_input_sets_the_status(cuda):
    d = 64
    rng = np.random.default_rng(0)
    _, pool = random_pool(rng, 3, 2, d, cuda)
    q = torch.randn(2, 4, d, device=cuda).to(torch.bfloat16)
    table = i32([[0, 1], [2, 7]], cuda)
    for lens, max_len, word in (([32, 32], 32, 0x203), ([33, 4], 32, 0x202), ([20, 3], 16, 0x202), ([32, 16], 32, 0)):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        o = kv4_attention(q, pool, i32(lens, cuda), table, max_len=max_len, status=status)
        assert int(status.item()) == word and torch.isfinite(o).all()
    for start in ([0, 3, 2], [-1, 1, 2], [0, 1, 9]):  # rows out of range: nothing of theirs is written
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        kv4_attention(q, pool, i32([20, 10], cuda), table, q_start=i32(start, cuda), status=status)
        assert int(status.item()) == 0x202


def test_attention_strides_streams_and_repeats(cuda):
    """Strided and unaligned q and out, another stream than the current one,
    and the same bits from every run."""
    rng = np.random.default_rng(9)
    heads, n_kv, d = 12, 3, 64
    side = torch.cuda.Stream(cuda)
    args, want = check_attention(cuda, rng, "f16", heads, n_kv, d, [5000, 77, 513], stream=side)
    q = args[0]
    for _ in range(3):
        assert torch.equal(kv4_attention(*args), want)
    wide = torch.zeros(3, heads, d + 1, dtype=torch.float16, device=cuda)[:, :, 1:]
    wide.copy_(q)
    out = torch.zeros(heads, 3, d + 1, dtype=torch.float16, device=cuda)[:, :, 1:].transpose(0, 1)
    kv4_attention(wide, *args[1:], out=out)
    assert torch.equal(out, want)
    # joined splits may differ from one pass only by float32 sums: both are within the bound, and repeat
    close = kv4_attention(*args, max_len=5000)
    assert torch.equal(close, kv4_attention(*args, max_len=5000))


def test_attention_in_graphs(cuda):
    """Captured once, replayed on new contents; two captured graphs (each with
    its own scratch) replayed at the same time on two streams."""
    rng = np.random.default_rng(12)
    args, _ = check_attention(cuda, rng, "bf16", 8, 2, 64, [4000, 900])
    q, pool, lens, table = args
    sets = [tuple(t.clone() for t in args) for _ in range(2)]
    outs, graphs = [], []
    for s in sets:
        out = torch.empty_like(q)
        kv4_attention(*s, out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv4_attention(*s, out=out)
        outs.append(out)
        graphs.append(g)
    for k in range(3):
        for i, s in enumerate(sets):
            s[0].copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(10 * k + i)).to(q.dtype))
            s[2].copy_(i32([4000 - 700 * k - i, 900 - 13 * k], cuda))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(cuda) for _ in range(2)]
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, out in zip(sets, outs):
            assert torch.equal(out, kv4_attention(*s))


def test_pool_past_32_bit_offsets(cuda):
    """Blocks whose bytes lie past 2^32 of the pool."""
    n_kv, d, blocks = 2, 128, 1_000_000  # 4.6 GB
    pool = torch.empty(blocks, n_kv, 18 * d, dtype=torch.uint8, device=cuda)
    table = i32([[blocks - 1, 3, blocks - 2]], cuda)
    n = 41
    k = torch.randn(n, n_kv, d, device=cuda).to(torch.bfloat16)
    v = torch.randn(n, n_kv, d, device=cuda).to(torch.bfloat16)
    zero, pos = i32(np.zeros(n), cuda), i32(np.arange(n), cuda)
    kv4_append(pool, k, v, pos, table, seq=zero)
    got_k, got_v = kv4_read(pool, pos, table, seq=zero, dtype=torch.float32)
    hk, hv = R.held(f64(k)), R.held(f64(v))
    assert np.array_equal(f64(got_k), hk) and np.array_equal(f64(got_v), hv)
    q = torch.randn(1, 4, d, device=cuda).to(torch.bfloat16)
    o = kv4_attention(q, pool, i32([n], cuda), table)
    want, mass, size = R.attention(f64(q), hk, hv, d ** -0.5)
    assert (np.abs(f64(o) - want) <= R.attention_bound(want, mass, size, n, d, 2.0 ** -8, np.abs(hv).max())).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("f16", 128)])
def test_prompt_then_tokens(cuda, dtype, d):
    """As a model runs them: a prompt's chunks, then tokens one by one, each
    appended and attended, two sequences in one batch, against the definition
    fed with the held keys and values."""
    t = TYPES[dtype]
    heads, n_kv, bps = 8, 2, 5
    rng = np.random.default_rng(d)
    table = rng.permutation(2 * bps).reshape(2, bps)
    table_d = i32(table, cuda)
    pool, status = new_kv4_pool(2 * bps, n_kv, d, cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    cos, sin = angles(16 * bps, d, cuda)
    gen = torch.Generator().manual_seed(d)
    past = [(np.zeros((0, n_kv, d)), np.zeros((0, n_kv, d))) for _ in range(2)]
    lens = [0, 0]
    for rows in ([18, 3], [9, 0], [1, 1], [1, 1], [1, 1], [4, 30], [1, 1]):
        n = sum(rows)
        seq = np.repeat([0, 1], rows)
        pos = np.concatenate([np.arange(a, a + r) for a, r in zip(lens, rows)])
        lens = [a + r for a, r in zip(lens, rows)]
        q, k, v = ((2 * torch.randn(n, h, d, generator=gen)).to(t).to(cuda) for h in (heads, n_kv, n_kv))
        turned = kv4_append(pool, k, v, i32(pos, cuda), table_d, seq=i32(seq, cuda), q=q, cos=cos, sin=sin,
                            status=status)
        start = None if rows == [1, 1] else i32(np.concatenate([[0], np.cumsum(rows)]), cuda)
        out = kv4_attention(turned, pool, i32(lens, cuda), table_d, q_start=start, status=status)
        check_status(status)
        hk, hv = R.held(R.turned(f64(k), f64(cos)[pos], f64(sin)[pos], False)), R.held(f64(v))
        for s in (0, 1):
            mine = seq == s
            past[s] = tuple(np.concatenate([p, x[mine]]) for p, x in zip(past[s], (hk, hv)))
            if mine.any():
                want, mass, size = R.attention(f64(turned)[mine], *past[s], d ** -0.5)
                bound = R.attention_bound(want, mass, size, lens[s], d, torch.finfo(t).eps / 2,
                                          np.abs(past[s][1]).max())
                assert (np.abs(f64(out)[mine] - want) <= bound).all()
