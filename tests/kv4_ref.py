"""The 4-bit cache and its operators from their definitions, in 64 bits
(numpy, test infrastructure)."""

from __future__ import annotations

import numpy as np

#: value of every scale byte the cache writes (0 .. 0xE1)
SCALES = np.array([b / 8 * 2.0 ** -14 for b in range(8)] +
                  [(1 + b % 8 / 8) * 2.0 ** (b // 8 - 15) for b in range(8, 0xE2)])


def held(x):
    """What the cache holds for rows x [..., d] (float64): groups of 16."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], -1, 16)
    a = np.where(np.isnan(g), 0.0, np.abs(g)).max(-1, keepdims=True)
    s = SCALES[np.minimum(np.searchsorted(SCALES * 7, a), SCALES.size - 1)]
    with np.errstate(invalid="ignore", divide="ignore"):
        n = np.clip(np.rint(np.where(s > 0, g / np.where(s > 0, s, 1.0), 0.0)), -7, 7)
    return (np.where(np.isnan(n), 0.0, n) * s).reshape(x.shape)


def turned(x, cos, sin, interleaved):
    """x [n, heads, d] turned by angles [n, r / 2] (float64)."""
    x = np.array(x, np.float64)
    r = 2 * cos.shape[1]
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    z = (x[..., lo] + 1j * x[..., hi]) * (cos.astype(np.float64) + 1j * sin.astype(np.float64))[:, None]
    x[..., lo], x[..., hi] = z.real, z.imag
    return x


def k_bytes(d, r, dim):
    """(byte of the code, low or high nibble, byte of the scale) of K, slot r, dim."""
    h, t, w = dim // 64, dim % 64 // 16, dim % 16
    unit = (h * 8 + r % 8) * 4 + t
    return unit * 16 + r // 8 * 8 + w // 2, w % 2, 8 * d + unit * 2 + r // 8


def v_bytes(d, r, dim):
    h, g, q, w = dim // 64, dim % 64 // 8, dim % 8 // 4, dim % 4
    t, p, e = r % 8 // 2, r // 8, r % 2
    code = 9 * d + (((((h * 8 + g) * 4 + t) * 2 + p) * 2 + q) * 2 + e) * 2 + w // 2
    return code, w % 2, 17 * d + (((h * 4 + dim % 64 // 16) * 4 + t) * 2 + p) * 2 + e


def page_values(pool, d):
    """uint8 [blocks, n_kv, 18 d] -> K, V [blocks, n_kv, 16, d] float64."""
    out = []
    table = np.concatenate([SCALES, np.full(256 - SCALES.size, np.nan)])
    for where in (k_bytes, v_bytes):
        idx = np.array([[where(d, r, i) for i in range(d)] for r in range(16)])
        code = pool[:, :, idx[..., 0]] >> (4 * idx[..., 1]).astype(np.uint8)
        out.append(((code & 15).astype(np.float64) - 8) * table[pool[:, :, idx[..., 2]]])
    return out


def sequence(pages, table_row, length):
    """Rows 0 .. length - 1 of a sequence: [length, n_kv, d]."""
    p = np.arange(length)
    return pages[table_row[p // 16], :, p % 16]


def attention(q, k, v, scale):
    """Rows q [n, heads, d], the last n positions of k, v [length, n_kv, d].
    Returns (out, sum of p |v|, largest sum of |q k| of a score), float64."""
    n, heads, d = q.shape
    length, n_kv = k.shape[:2]
    out, mass, size = np.zeros((n, heads, d)), np.zeros((n, heads, d)), np.zeros((n, heads, 1))
    for h in range(heads):
        g = h // (heads // n_kv)
        s = q[:, h] @ k[:, g].T * scale
        s[np.arange(length)[None] > length - n + np.arange(n)[:, None]] = -np.inf
        for j in range(n):
            if not np.isfinite(s[j]).any():
                continue
            p = np.exp(s[j] - s[j].max())
            p /= p.sum()
            out[j, h], mass[j, h] = p @ v[:, g], p @ np.abs(v[:, g])
            seen = np.isfinite(s[j])
            size[j, h] = (np.abs(q[j, h]) @ np.abs(k[seen, g]).T).max() * scale
    return out, mass, size


def attention_bound(out, mass, size, length, d, half_step, vmax):
    """How far the kernel may be off.  ``half_step``: finfo(type).eps / 2.

    * the result is rounded once: half_step |o|;
    * each probability is rounded to a half: 2^-11 of sum p |v|;
    * a score is a float32 sum of d products, scaled once, minus the maximum:
      off by (d + 3) 2^-24 of sum |q k|, which shifts log2 p by that times
      log2(e); with the maximum's own, p changes by twice that share, and so
      does the sum of p it is divided by: 4 in all;
    * 2^x is good to 2^-22, and its argument (a difference of scores of at most
      `size` each) is rounded: 3 * 2^-24 size, in numerator and divisor;
    * float32 sums over the positions: a chain of length / 16 products of 16
      and the rescaling after each, (length / 16 + 64) 2^-23 of sum p |v|,
      again for numerator and divisor;
    * a probability is a half with a factor of at least 2^10 that the row's sum
      (at least that factor) carries too; halves below 2^-14 are 2^-24 apart, so
      it is off by up to 2^-25 / 2^10 = 2^-35, at each of `length` positions with
      |v| <= vmax;
    * an fp16 result's rounding is off by up to 2^-25 however small it is.
    """
    low = length * 2.0 ** -35 * vmax + (2.0 ** -25 if half_step == 2.0 ** -11 else 0.0)
    share = 2.0 ** -11 + 4 * (d + 6) * 2.0 ** -24 * size + 2.0 ** -20 + 2 * (length / 16 + 64) * 2.0 ** -23
    return half_step * np.abs(out) + share * (1 + half_step) * mass + low + 1e-30
