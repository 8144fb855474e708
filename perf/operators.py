"""The serving operators over a 4-bit KV cache, and the logits adjustment, as cases to measure.

Three operators, each in a plain form (elementary torch operations) and as the
calls a user makes:

* ``append``    rotary positions on the query and key rows of a packed
  projection, the key and value rows quantised to 4 bits and written to a
  paged cache, then read back as values (``kv4_append``, ``kv4_read``);
* ``attention`` causal attention over that cache, one row a sequence (decode)
  or several (a prompt's chunk) (``kv4_attention``);
* ``logits``    repetition, presence and frequency penalties, biases and token
  masks on a batch of logits (``adjust_logits``).

The cache's format: a position's row of one kv head is cut into groups of 16
dims.  A group's scale s is the smallest number >= amax / 7 with 5 exponent
and 3 mantissa bits (its byte b is the half with the bits ``b << 7``), at most
9216; a value x is held as clamp(round(x / s), -7, 7), plus 8, in a nibble.  A
page holds 16 positions of one kv head in 18 d bytes: K codes (8 d), K scales
(d), V codes (8 d), V scales (d), in the orders ``_keys`` and ``_values`` read.
"""

from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
TOP_SCALE = 9216.0


# ---- cases ----------------------------------------------------------------

def _attention(name, dtype, heads, kv_heads, d, batch, min_len, max_len, rows=1):
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "d": d,
            "batch": batch, "min_len": min_len, "max_len": max_len, "rows": rows}


def _append(name, dtype, heads, kv_heads, d, batch, min_len, max_len, rows, rope, rotary):
    return {"name": name, "op": "append", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "d": d,
            "batch": batch, "min_len": min_len, "max_len": max_len, "rows": rows, "rope": rope, "rotary": rotary}


def _logits(name, batch, vocab, history, biases, masked):
    return {"name": name, "op": "logits", "batch": batch, "vocab": vocab, "history": history, "biases": biases,
            "masked": masked}


def listed():
    return [
        # one chat at the end of this model's context: a layer's call, all latency
        _attention("attend one row, context 512", "bf16", 16, 4, 64, 1, 512, 512),
        # a full serving wave of this model: ragged rows, one slot idle
        _attention("attend wave of 256", "bf16", 16, 4, 64, 256, 0, 511),
        # one very long conversation on a model with wider heads
        _attention("attend one row, 131071 positions", "bf16", 32, 8, 128, 1, 131071, 131071),
        # a serving batch of long conversations: the cache read bounds it
        _attention("attend 32 rows to 16384", "f16", 32, 8, 128, 32, 1001, 16384),
        # this model's prompt pass: one prompt that fills the context
        _attention("attend prompt of 512", "bf16", 16, 4, 64, 1, 512, 512, rows=512),
        # chunks of long prompts of four requests in one pass, ragged
        _attention("attend 4 chunks to 8191", "f16", 32, 8, 128, 4, 2049, 8191, rows=512),
        # one token of one chat, a layer's call
        _append("append one row", "bf16", 16, 4, 64, 1, 512, 512, 1, "half", 64),
        # this model's prompt pass: 512 rows of several prompts
        _append("append 512 rows", "bf16", 16, 4, 64, 7, 32, 448, 100, "half", 64),
        # a large prompt pass of a model that rotates half of each head, pairs interleaved
        _append("append 8192 rows", "f16", 32, 8, 128, 9, 1001, 16384, 1821, "interleaved", 64),
        # one sampled chat, no mask: all latency
        _logits("logits of one row", 1, 32000, 300, 3, 0.0),
        # a sampled wave of this model under grammars that allow few tokens
        _logits("logits of 256 rows, grammar", 256, 32000, 511, 16, 0.98),
        # a large vocabulary of odd size, long histories, a few banned tokens
        _logits("logits of 65 rows of 100003", 65, 100003, 4096, 300, 0.001),
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def _heads(rng):
    d = rng.choice((64, 128))
    kv = rng.choice((1, 2, 3, 4, 5, 8))
    return rng.choice(tuple(TYPES)), kv * rng.choice((1, 2, 3, 4, 5, 7, 8)), kv, d


def draw(rng):
    op = rng.choice(("attention", "attention", "append", "logits"))
    if op == "logits":
        batch, vocab = _log(rng, 1, 256), _log(rng, 500, 131072)
        batch = max(1, min(batch, 256 * 32000 // vocab))
        c = _logits("", batch, vocab, _log(rng, 1, 4096), _log(rng, 1, min(300, vocab)),
                    rng.choice((0.0, 0.001, 0.3, 0.98)))
    elif op == "append":
        dtype, heads, kv, d = _heads(rng)
        heads, batch = min(heads, 32), _log(rng, 1, 64)
        heads -= heads % kv
        rows = _log(rng, 1, max(1, 4096 // batch))
        max_len = _log(rng, rows, 16384)
        c = _append("", dtype, heads, kv, d, batch, rng.randint(min(rows, max_len), max_len), max_len, rows,
                    rng.choice(("half", "interleaved")), rng.choice((d, d, d // 2, d // 4 * 3, 2)))
    else:
        dtype, heads, kv, d = _heads(rng)
        if rng.random() < 0.6:
            batch, rows = _log(rng, 1, 256), 1
            room = 32 * 16384 * 8 * 64 // (batch * kv * d)
            max_len = min(_log(rng, 1, 131072), room)
        else:
            batch, rows = _log(rng, 1, 8), _log(rng, 2, 512)
            heads = min(heads, 32)
            heads -= heads % kv
            room = 32 * 128 * 4 * 512 * 4096 // (heads * d * batch * rows)
            max_len = min(_log(rng, rows, 16384), max(room, rows))
        c = _attention("", dtype, heads, kv, d, batch, rng.randint(0, max_len), max_len, rows)
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, in an order that mixes short and long."""
    step = next(s for s in range(max(1, int(n * 0.618)), 2 * n + 2) if math.gcd(s, n) == 1)
    return [hi if n == 1 else lo + (hi - lo) * (i * step % n) // (n - 1) for i in range(n)]


def _sizes(case):
    """(lengths, rows) of each sequence; a sequence's rows are its last positions."""
    lens = _spread(case["min_len"], case["max_len"], case["batch"])
    if case["op"] == "attention" and case["rows"] == 1:
        return lens, [1] * len(lens)
    rows = _spread(max(1, case["rows"] // 4), case["rows"], case["batch"])
    return lens, [min(r, n) for r, n in zip(rows, lens)]


def work(case):
    if case["op"] == "logits":
        b, v = case["batch"], case["vocab"]
        mask = b * ((v + 31) // 32) * 4 if case["masked"] else 0
        return {"bytes": 8 * b * v + 4 * b * case["history"] + 8 * b * case["biases"] + mask, "flops": 4 * b * v}
    lens, rows = _sizes(case)
    h, kv, d = case["heads"], case["kv_heads"], case["d"]
    n = sum(rows)
    if case["op"] == "append":
        held = n * kv * d * 9 // 8  # codes and scales of K and V
        # q, k, v read, q written; the cache's rows written, read and given back as values; angles
        size = 2 * n * d * (2 * h + 2 * kv) + 2 * held + 4 * n * kv * d + 4 * n * case["rotary"]
        return {"bytes": size, "flops": 6 * n * case["rotary"] * (h + kv) // 2 + 4 * n * kv * d}
    seen = sum(max(0, ln - r + j + 1) for ln, r in zip(lens, rows) for j in range(r))
    size = sum(lens) * kv * d * 9 // 8 + 4 * n * h * d + 4 * sum((ln + PAGE - 1) // PAGE for ln in lens)
    return {"bytes": size, "flops": 4 * d * h * seen}


# ---- inputs ---------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _table(lens, gen, spare=3):
    """Pages of sequences of `lens` positions, in any order: (table, pages in the pool)."""
    pages = [(n + PAGE - 1) // PAGE for n in lens]
    total = sum(pages) + spare
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(1, max(pages)), dtype=torch.int32, device="cuda")
    have = torch.arange(table.shape[1], device="cuda")[None, :] < torch.tensor(pages, device="cuda")[:, None]
    table[have] = order[:sum(pages)]
    return table, total


def _channels(d, gen):
    """Key channels of unlike size, a few far larger than the rest."""
    c = torch.exp(0.5 * torch.randn(d, generator=gen, device="cuda"))
    return c * torch.where(torch.rand(d, generator=gen, device="cuda") < 0.03, 6.0, 1.0)


def _fill(pool, d, gen):
    """A pool of normal keys and values, held as the cache holds them."""
    chan = _channels(d, gen)
    for lo in range(0, pool.shape[0], 2048):
        part = pool[lo:lo + 2048]
        n, kv = part.shape[:2]
        k = torch.randn(n, kv, PAGE, d, generator=gen, device="cuda") * chan
        v = torch.randn(n, kv, PAGE, d, generator=gen, device="cuda")
        (kc, ks), (vc, vs) = _quantised(k), _quantised(v)
        nh = d // 64
        # K codes [h][g][t][e][8 bytes]: position 8e + g, dims 64h + 16t ..
        kc = kc.view(n, kv, 2, 8, nh, 4, 8, 2).permute(0, 1, 4, 3, 5, 2, 6, 7)
        part[:, :, :8 * d] = (kc[..., 0] + 16 * kc[..., 1]).to(torch.uint8).reshape(n, kv, -1)
        part[:, :, 8 * d:9 * d] = ks.view(n, kv, 2, 8, nh, 4).permute(0, 1, 4, 3, 5, 2).reshape(n, kv, -1)
        # V codes [h][g][t][p][q][e][2 bytes]: position 8p + 2t + e, dims 64h + 8g + 4q ..
        vc = vc.view(n, kv, 2, 4, 2, nh, 8, 2, 2, 2).permute(0, 1, 5, 6, 3, 2, 7, 4, 8, 9)
        part[:, :, 9 * d:17 * d] = (vc[..., 0] + 16 * vc[..., 1]).to(torch.uint8).reshape(n, kv, -1)
        # V scales [h][G][t][p][e]: position 8p + 2t + e, dims 64h + 16G ..
        part[:, :, 17 * d:] = vs.view(n, kv, 2, 4, 2, nh, 4).permute(0, 1, 5, 6, 3, 2, 4).reshape(n, kv, -1)


def prepare(case, seed):
    gen = _gen(seed)
    if case["op"] == "logits":
        b, v, cap = case["batch"], case["vocab"], case["history"]
        logits = 3.0 * torch.randn(b, v, generator=gen, device="cuda")
        # text repeats itself: tokens by a steep law, some in every row
        u = torch.rand(b, cap, generator=gen, device="cuda")
        history = (u.pow(4) * v).to(torch.int32).clamp_(max=v - 1)
        hist_len = torch.randint(0, cap + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        prompt_len = (hist_len * torch.rand(b, generator=gen, device="cuda")).to(torch.int32)
        pick = torch.rand(b, v, generator=gen, device="cuda").topk(case["biases"], dim=1).indices
        st = {"op": "logits", "logits": logits, "history": history, "hist_len": hist_len, "prompt_len": prompt_len,
              "rep": 1.0 + 0.1 * torch.randint(0, 4, (b,), generator=gen, device="cuda"),
              "presence": 0.5 * torch.randint(0, 3, (b,), generator=gen, device="cuda"),
              "frequency": 0.25 * torch.randint(0, 3, (b,), generator=gen, device="cuda"),
              "bias_ids": pick.to(torch.int32).contiguous(),
              "bias_values": 2.0 * torch.randn(b, case["biases"], generator=gen, device="cuda"),
              "bias_len": torch.randint(0, case["biases"] + 1, (b,), generator=gen, device="cuda", dtype=torch.int32),
              "allowed": None}
        if case["masked"]:
            words = (v + 31) // 32
            bits = torch.rand(b, words, 32, generator=gen, device="cuda") >= case["masked"]
            place = torch.arange(32, device="cuda")
            whole = (bits.to(torch.int64) << place).sum(-1)
            st["allowed"] = torch.where(whole >= 1 << 31, whole - (1 << 32), whole).to(torch.int32)
        return st
    dtype, h, kv, d = TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["d"]
    lens, rows = _sizes(case)
    n = sum(rows)
    table, total = _table(lens, gen)
    if case["op"] == "append":
        qkv = torch.randn(n, (h + 2 * kv) * d, generator=gen, device="cuda")
        qkv[:, h * d:(h + kv) * d] *= _channels(d, gen).repeat(kv)
        qkv = qkv.to(dtype)
        pos = torch.cat([torch.arange(ln - r, ln) for ln, r in zip(lens, rows)]).to(torch.int32).cuda()
        seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows)).to(torch.int32).cuda()
        at = torch.arange(case["max_len"], dtype=torch.float64)[:, None]
        ang = at * 10000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])
        return {"op": "append", "q": qkv[:, :h * d].view(n, h, d), "k": qkv[:, h * d:(h + kv) * d].view(n, kv, d),
                "v": qkv[:, (h + kv) * d:].view(n, kv, d), "pos": pos, "seq": seq, "table": table,
                "cos": ang.cos().float().cuda(), "sin": ang.sin().float().cuda(), "rope": case["rope"],
                "pool": torch.zeros(total, kv, 18 * d, dtype=torch.uint8, device="cuda")}
    pool = torch.empty(total, kv, 18 * d, dtype=torch.uint8, device="cuda")
    _fill(pool, d, gen)
    st = {"op": "attention", "q": torch.randn(n, h, d, generator=gen, device="cuda").to(dtype), "pool": pool,
          "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "q_start": None,
          "max_rows": 1}
    if case["rows"] > 1:
        st["q_start"] = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
        st["max_rows"] = max(rows)
    return st


# ---- the plain forms ------------------------------------------------------

def _quantised(x):
    """Rows of x in groups of 16: (codes 1..15, scale bytes), x in 32 or 64 bits."""
    g = x.unflatten(-1, (-1, 16))
    want = g.abs().amax(-1) / 7
    _, e = torch.frexp(want)
    step = torch.ldexp(torch.ones_like(want), e.clamp(min=-13) - 4)  # of numbers with 3 mantissa bits near `want`
    s = ((want / step).ceil() * step).clamp(max=TOP_SCALE)
    codes = torch.where(s[..., None] > 0, g / s[..., None], 0.0).round().clamp(-7, 7) + 8
    return codes.flatten(-2).to(torch.int32), (s.to(torch.float16).view(torch.int16) >> 7).to(torch.uint8)


def _scale(b):
    return (b.to(torch.int16) << 7).view(torch.float16).float()


def _nibbles(b):
    return torch.stack((b & 15, b >> 4), -1).float() - 8


def _keys(pages, d):
    """[B, P, kv, 18 d] -> keys [B, kv, 16 P, d]."""
    b, p, kv, nh = *pages.shape[:3], d // 64
    c = _nibbles(pages[..., :8 * d].reshape(b, p, kv, nh, 8, 4, 2, 8)).flatten(-2)
    s = _scale(pages[..., 8 * d:9 * d].reshape(b, p, kv, nh, 8, 4, 2, 1))
    return (c * s).permute(0, 2, 1, 6, 4, 3, 5, 7).reshape(b, kv, PAGE * p, d)


def _values(pages, d):
    """[B, P, kv, 18 d] -> values [B, kv, 16 P, d]."""
    b, p, kv, nh = *pages.shape[:3], d // 64
    c = _nibbles(pages[..., 9 * d:17 * d].reshape(b, p, kv, nh, 8, 4, 2, 2, 2, 2)).flatten(-2)
    c = c.permute(0, 2, 1, 6, 5, 8, 3, 4, 7, 9).reshape(b, kv, PAGE * p, d // 16, 16)
    s = _scale(pages[..., 17 * d:].reshape(b, p, kv, nh, 4, 4, 2, 2))
    s = s.permute(0, 2, 1, 6, 5, 7, 3, 4).reshape(b, kv, PAGE * p, d // 16, 1)
    return (c * s).flatten(-2)


def _rotated(x, cos, sin, rope):
    """The first 2 * cos.shape[-1] dims of each head turned by the row's angles."""
    r = 2 * cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    if rope == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat((a * c - b * s, a * s + b * c, x[..., r:]), -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat((torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2), x[..., r:]), -1)


def _plain_append(st):
    # in 64 bits: a rotated key next to the border of two codes belongs to one of them
    pos, dtype = st["pos"].long(), st["q"].dtype
    cos, sin = st["cos"][pos].double(), st["sin"][pos].double()
    q = _rotated(st["q"].double(), cos, sin, st["rope"]).to(dtype)
    kc, ks = _quantised(_rotated(st["k"].double(), cos, sin, st["rope"]))
    vc, vs = _quantised(st["v"].double())
    k = (kc.unflatten(-1, (-1, 16)) - 8).float() * _scale(ks)[..., None]
    v = (vc.unflatten(-1, (-1, 16)) - 8).float() * _scale(vs)[..., None]
    return {"q": q, "k": k.flatten(-2).to(dtype), "v": v.flatten(-2).to(dtype)}


def _plain_attention(st):
    q, d = st["q"].float(), st["q"].shape[-1]
    pages = st["pool"][st["table"].long()]
    k, v = _keys(pages, d), _values(pages, d)
    b, kv, length = k.shape[:3]
    lens = st["lens"].long()
    if st["q_start"] is None:
        q, rows = q[:, None], torch.ones_like(lens)
    else:
        start = st["q_start"].long()
        rows = start[1:] - start[:-1]
        at = (start[:-1, None] + torch.arange(st["max_rows"], device=q.device)).clamp(max=q.shape[0] - 1)
        q = q[at]
    r = q.shape[1]
    j = torch.arange(r, device=q.device)
    last = (lens - rows)[:, None] + j  # the last position that a row sees
    q = q.unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [b, kv, group * rows, d]
    s = (q @ k.transpose(-1, -2) / math.sqrt(d)).unflatten(2, (-1, r))
    sees = torch.arange(length, device=q.device) <= last[..., None]
    s = s.masked_fill(~sees[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    e = (s - top).exp()
    o = e.flatten(2, 3) @ v / e.sum(-1).clamp(min=1e-30).flatten(2, 3)[..., None]
    o = o.unflatten(2, (-1, r)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[j < rows[:, None]].to(st["q"].dtype)


def _plain_logits(st):
    x, v = st["logits"], st["logits"].shape[1]
    ids = st["history"].long()
    at = torch.arange(ids.shape[1], device=x.device)
    held = at < st["hist_len"][:, None]
    made = held & (at >= st["prompt_len"][:, None])
    zero = torch.zeros_like(x)
    seen, count = zero.scatter_add(1, ids, held.float()), zero.scatter_add(1, ids, made.float())
    rep = st["rep"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (st["frequency"][:, None] * count + st["presence"][:, None] * (count > 0))
    n = torch.arange(st["bias_ids"].shape[1], device=x.device) < st["bias_len"][:, None]
    x = x + zero.scatter_add(1, st["bias_ids"].long(), torch.where(n, st["bias_values"], 0.0))
    if st["allowed"] is not None:
        bits = (st["allowed"][..., None] >> torch.arange(32, device=x.device)) & 1
        x = x.masked_fill(bits.flatten(1)[:, :v] == 0, -math.inf)
    return x


def run(st):
    if own:
        if st["op"] == "append":
            from transformer_b200.kv4 import kv4_append, kv4_read
            q = kv4_append(st["pool"], st["k"], st["v"], st["pos"], st["table"], seq=st["seq"], q=st["q"],
                           cos=st["cos"], sin=st["sin"], interleaved=st["rope"] == "interleaved")
            k, v = kv4_read(st["pool"], st["pos"], st["table"], seq=st["seq"], dtype=st["k"].dtype)
            return {"q": q, "k": k, "v": v}
        if st["op"] == "attention":
            from transformer_b200.kv4 import kv4_attention
            return kv4_attention(st["q"], st["pool"], st["lens"], st["table"], q_start=st["q_start"],
                                 max_rows=st["max_rows"])
        from transformer_b200.generate import adjust_logits
        return adjust_logits(st["logits"], history=st["history"], hist_len=st["hist_len"],
                             prompt_len=st["prompt_len"], rep_penalty=st["rep"], presence=st["presence"],
                             frequency=st["frequency"], bias_ids=st["bias_ids"], bias_values=st["bias_values"],
                             bias_len=st["bias_len"], allowed=st["allowed"])
    if st["op"] == "append":
        return _plain_append(st)
    return _plain_attention(st) if st["op"] == "attention" else _plain_logits(st)


# ---- the definitions, in 64 bits ------------------------------------------

def _grid():
    """Every scale, by its byte."""
    tiny = [b / 8 * 2.0 ** -14 for b in range(8)]
    return tiny + [(1 + b % 8 / 8) * 2.0 ** (b // 8 - 15) for b in range(8, 226)]


def _exact_held(x):
    """What the cache holds for rows x."""
    grid = torch.tensor(_grid(), dtype=torch.float64, device=x.device)
    g = x.reshape(*x.shape[:-1], -1, 16)
    want = g.abs().max(-1, keepdim=True).values / 7
    s = grid[torch.searchsorted(grid, want).clamp(max=grid.numel() - 1)]
    y = g / s.clamp(min=2.0 ** -17)
    n = torch.floor(y + 0.5)
    n = n - ((n - y == 0.5) & (n % 2 != 0)).double()
    return (n.clamp(-7, 7) * s).reshape(x.shape)


def _exact_append(st):
    pos = st["pos"].long()
    turn = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, None]
    r = 2 * turn.shape[-1]

    def rotated(x):
        x = x.double().clone()
        lo, hi = (slice(0, r // 2), slice(r // 2, r)) if st["rope"] == "half" else (slice(0, r, 2), slice(1, r, 2))
        z = torch.complex(x[..., lo], x[..., hi]) * turn
        x[..., lo], x[..., hi] = z.real, z.imag
        return x

    return {"q": rotated(st["q"]), "k": _exact_held(rotated(st["k"])), "v": _exact_held(st["v"].double())}


def _exact_rows(pool, table, length, d):
    """Keys and values [length, kv, d] of one sequence, byte by byte from the page's layout."""
    grid = torch.tensor(_grid() + [math.nan] * 30, dtype=torch.float64, device=pool.device)
    p = torch.arange(length, device=pool.device)
    page = pool[table[p // PAGE].long()]  # [length, kv, 18 d]
    i = torch.arange(d, device=pool.device)
    r = (p % PAGE)[:, None]
    h, w = i // 64, i % 64
    unit = (h * 8 + r % 8) * 4 + w // 16
    code = unit * 16 + r // 8 * 8 + w % 16 // 2
    scale = 8 * d + unit * 2 + r // 8
    kv = page.shape[1]

    def at(where):
        return torch.gather(page, 2, where[:, None].expand(-1, kv, -1)).long()

    k = ((at(code) >> 4 * (i % 2)) % 16 - 8) * grid[at(scale)]
    t, half, odd = r % 8 // 2, r // 8, r % 2
    code = 9 * d + (((((h * 8 + w // 8) * 4 + t) * 2 + half) * 2 + w % 8 // 4) * 2 + odd) * 2 + w % 4 // 2
    scale = 17 * d + (((h * 4 + w // 16) * 4 + t) * 2 + half) * 2 + odd
    v = ((at(code) >> 4 * (i % 2)) % 16 - 8) * grid[at(scale)]
    return k, v


def _exact_attention(st):
    q, d = st["q"].double(), st["q"].shape[-1]
    out = torch.zeros_like(q)
    lens = st["lens"].tolist()
    start = list(range(len(lens) + 1)) if st["q_start"] is None else st["q_start"].tolist()
    for b, n in enumerate(lens):
        rows = start[b + 1] - start[b]
        if n < 1 or rows < 1:
            continue
        k, v = _exact_rows(st["pool"], st["table"][b], n, d)
        group = q.shape[1] // k.shape[1]
        for g in range(k.shape[1]):
            mine = q[start[b]:start[b + 1], g * group:(g + 1) * group]
            s = torch.einsum("jhd,ld->jhl", mine, k[:, g]) / math.sqrt(d)
            hidden = torch.arange(n, device=q.device)[None] > n - rows + torch.arange(rows, device=q.device)[:, None]
            p = torch.softmax(s.masked_fill(hidden[:, None], -math.inf), -1)
            out[start[b]:start[b + 1], g * group:(g + 1) * group] = torch.einsum("jhl,ld->jhd", p, v[:, g])
    return out


def _exact_logits(st):
    out = st["logits"].double().clone()
    v = out.shape[1]
    for b in range(out.shape[0]):
        ids = st["history"][b, :st["hist_len"][b]].long()
        count = torch.bincount(ids[st["prompt_len"][b]:], minlength=v).double()
        x, rep = out[b], st["rep"][b].double()
        old = torch.unique(ids)
        x[old] = torch.where(x[old] > 0, x[old] / rep, x[old] * rep)
        x -= st["frequency"][b].double() * count
        x -= st["presence"][b].double() * (count > 0)
        n = int(st["bias_len"][b])
        x[st["bias_ids"][b, :n].long()] += st["bias_values"][b, :n].double()
        if st["allowed"] is not None:
            token = torch.arange(v, device=out.device)
            x[(st["allowed"][b][token // 32] >> (token % 32)) & 1 == 0] = -math.inf
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if st["op"] == "append":
        return _exact_append(st)
    return _exact_attention(st) if st["op"] == "attention" else _exact_logits(st)
