"""GPU: the decode engine and the continuous batcher on 4-bit paged pools, and
requests with rules of their own on their logits.

A step is compared with the float32 oracle fed with the keys and values that
the device's pool holds (read back through kv4_read): what is left between
them is the bf16 decode's own error, the bound of every parity test here.  The
pool's rows are compared with the keys and values that the oracle computes on
the way: held values lie within half a scale (at most 8/7 of amax / 7) of what
the device quantised, which the parity bound separates from the oracle's."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import ATOL, RTOL, assert_logits_close
from oracle.ref_forward import CachedDecoder
from transformer_b200 import _lib
from transformer_b200.kv4 import kv4_read
from transformer_b200.multi_sm_decode import PAGE_TOKENS, DecodeEngine
from transformer_b200.serve import ContinuousBatcher

pytestmark = pytest.mark.gpu


class Given(np.ndarray):
    """An array that keeps what it has; writes are noted instead."""

    def __setitem__(self, key, value):
        self.notes.append((key, np.array(value)))


def step_on_pool(P, cfg, eng, pool, row, tok, pos):
    """The oracle's step at `pos` over the keys and values in the device's pool;
    checks the row of `pos` in it.  Returns the logits."""
    dec = CachedDecoder(P, cfg, 1)
    at = torch.arange(pos + 1, dtype=torch.int32, device=eng.device)
    seq, table = torch.zeros_like(at), row[None].contiguous()
    for l in range(cfg.n_layers):
        for held, x in zip(kv4_read(pool[l], at, table, seq=seq, dtype=torch.float32), (dec.K, dec.V)):
            x[0, l, :, :pos + 1] = held.permute(1, 0, 2).cpu().numpy()
    dec.K, dec.V = dec.K.view(Given), dec.V.view(Given)
    dec.K.notes, dec.V.notes = [], []
    lg = dec.step([tok], [pos])[0]
    for x in (dec.K, dec.V):
        assert len(x.notes) == cfg.n_layers
        for (_, l, _, p), want in x.notes:
            held = np.asarray(x[0, l, :, p], np.float64)
            amax = np.abs(want.reshape(cfg.n_kv_heads, -1, 16)).max(-1, keepdims=True)
            half = (amax + ATOL + RTOL * amax) / 7 * (8 / 7) / 2
            off = np.abs(held - want).reshape(cfg.n_kv_heads, -1, 16)
            assert (off <= half + ATOL + RTOL * np.abs(want).reshape(off.shape)).all(), (l, float(off.max()))
    return lg


@pytest.fixture(scope="module")
def tiny4(engine_tiny):
    eng = DecodeEngine(engine_tiny.w, max_batch=64, kv_bits=4)
    yield eng
    eng.close()


@pytest.fixture(scope="module")
def big4(engine306):
    eng = DecodeEngine(engine306.w, max_batch=256, kv_bits=4)
    yield eng
    eng.close()


def _tables(rng, n, bps, dev, spare=3):
    t = rng.permutation(n * bps + spare)[:n * bps].reshape(n, bps).astype(np.int32)
    return torch.from_numpy(t).to(dev), n * bps + spare


def test_prompt_rows_then_steps_tiny(tiny4, params_tiny):
    """Ragged prompts of several sequences in one b2d_prefill_rows pass, an idle
    row among the decode steps that follow (the third replays a graph)."""
    from transformer_b200.config import CONFIG_TINY as cfg
    from transformer_b200.synth import params_f32
    P, eng, dev = params_f32(params_tiny), tiny4, tiny4.device
    rng = np.random.default_rng(77)
    lens = [1, 17, 40, 100, 16]
    table, nb = _tables(rng, len(lens), cfg.context_len // PAGE_TOKENS, dev)
    pool = eng.new_kv_pool(nb)
    prompts = [rng.integers(0, cfg.vocab_size, n).astype(np.int32) for n in lens]
    rows = [(i, p) for i, n in enumerate(lens) for p in range(n - 1)] + [(i, n - 1) for i, n in enumerate(lens)]
    tok = torch.tensor([int(prompts[i][p]) for i, p in rows], dtype=torch.int32, device=dev)
    pos = torch.tensor([p for _, p in rows], dtype=torch.int32, device=dev)
    lg = torch.zeros(len(lens), cfg.vocab_size, device=dev)
    nt = torch.zeros(len(lens), dtype=torch.int32, device=dev)
    eng.prefill_rows(tok, pos, pool, table[[i for i, _ in rows]].contiguous(), len(lens), lg, nt)
    eng.check_device()
    for i, n in enumerate(lens):
        assert_logits_close(lg[i].cpu().numpy(), step_on_pool(P, cfg, eng, pool, table[i], prompts[i][-1], n - 1))
    tok, pos = nt.clone(), torch.tensor(lens, dtype=torch.int32, device=dev)
    for k in range(4):
        pos[4] = -1 if k == 1 else lens[4] + k
        was, at = tok.clone(), pos.clone()
        eng.step_paged(tok, pos, pool, table, lg, nt)
        eng.check_device()
        for i in range(len(lens)):
            if at[i] >= 0:
                ref = step_on_pool(P, cfg, eng, pool, table[i], int(was[i]), int(at[i]))
                assert_logits_close(lg[i].cpu().numpy(), ref)
        tok.copy_(nt)
        pos += 1


@pytest.mark.parametrize("chunks", [[1], [37], [128], [20, 90, 1]])
def test_prompt_of_one_sequence_tiny(tiny4, params_tiny, chunks):
    from transformer_b200.config import CONFIG_TINY as cfg
    from transformer_b200.synth import params_f32
    P, eng = params_f32(params_tiny), tiny4
    rng = np.random.default_rng(sum(chunks))
    table, nb = _tables(rng, 1, cfg.context_len // PAGE_TOKENS, eng.device)
    pool, start = eng.new_kv_pool(nb), 0
    prompt = rng.integers(0, cfg.vocab_size, sum(chunks)).astype(np.int32)
    for c in chunks:
        lg = eng.prefill_paged(prompt[start:start + c], pool, table[0], start)
        start += c
        eng.check_device()
        ref = step_on_pool(P, cfg, eng, pool, table[0], prompt[start - 1], start - 1)
        assert_logits_close(lg.cpu().numpy(), ref)
        assert int(eng.next_tok[0]) == int(lg.argmax())
    used = table[0, :(start + PAGE_TOKENS - 1) // PAGE_TOKENS].long()
    rest = torch.ones(nb, dtype=torch.bool, device=eng.device)
    rest[used] = False
    assert torch.count_nonzero(pool[:, rest]) == 0


def test_306m_prompt_and_step(big4, params306_f32):
    """A 384-token prompt in one pass, then decode steps of a batch of 70."""
    from transformer_b200.config import CONFIG_306M as cfg
    eng, dev = big4, big4.device
    rng = np.random.default_rng(6)
    B = 70
    table, nb = _tables(rng, B, cfg.context_len // PAGE_TOKENS, dev)
    pool = eng.new_kv_pool(nb)
    prompt = rng.integers(0, cfg.vocab_size, 384).astype(np.int32)
    lg = eng.prefill_paged(prompt, pool, table[0])
    assert_logits_close(lg.cpu().numpy(), step_on_pool(params306_f32, cfg, eng, pool, table[0], prompt[-1], 383))
    tok = torch.from_numpy(rng.integers(0, cfg.vocab_size, B).astype(np.int32)).to(dev)
    pos = torch.zeros(B, dtype=torch.int32, device=dev)
    pos[0] = 384
    logits, nt = torch.zeros(B, cfg.vocab_size, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    for _ in range(3):
        was, at = tok.clone(), pos.clone()
        eng.step_paged(tok, pos, pool, table, logits, nt)
        tok.copy_(nt)
        pos += 1
    eng.check_device()
    for b in (0, 1, 69):
        ref = step_on_pool(params306_f32, cfg, eng, pool, table[b], int(was[b]), int(at[b]))
        assert_logits_close(logits[b].cpu().numpy(), ref)


def test_step_repeats_bit_for_bit(big4):
    from transformer_b200.config import CONFIG_306M as cfg
    eng, dev = big4, big4.device
    rng = np.random.default_rng(8)
    table, nb = _tables(rng, 8, cfg.context_len // PAGE_TOKENS, dev)
    pool = eng.new_kv_pool(nb)
    tok = torch.from_numpy(rng.integers(0, cfg.vocab_size, 8).astype(np.int32)).to(dev)
    pos = torch.arange(8, dtype=torch.int32, device=dev) * 0
    nt, out = torch.zeros(8, dtype=torch.int32, device=dev), []
    for _ in range(4):
        lg = torch.zeros(8, cfg.vocab_size, device=dev)
        eng.step_paged(tok, pos, pool, table, lg, nt)
        out.append((lg, pool.clone()))
    assert all(torch.equal(a, out[0][0]) and torch.equal(b, out[0][1]) for a, b in out[1:])


def test_pools_are_not_mixed_up(tiny4, engine_tiny_batched):
    dev = tiny4.device
    ints = torch.zeros(2, dtype=torch.int32, device=dev)
    table = torch.zeros(2, 8, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        tiny4.step_paged(ints, ints, engine_tiny_batched.new_kv_pool(4), table)
    with pytest.raises(ValueError):
        engine_tiny_batched.step_paged(ints, ints, tiny4.new_kv_pool(4), table)
    with pytest.raises(ValueError):
        DecodeEngine(tiny4.w, 2, kv_bits=8)
    assert tiny4.lib.b2d_workspace_kv_bits(tiny4.ws, 5) == _lib.B2D_ERR_INVALID_ARG
    assert tiny4.lib.b2d_workspace_kv_bits(None, 4) == _lib.B2D_ERR_INVALID_ARG


def test_bad_table_entries_set_the_status(tiny4):
    eng, dev = tiny4, tiny4.device
    pool = eng.new_kv_pool(4)
    ints = torch.zeros(2, dtype=torch.int32, device=dev)
    for entry in (4, -1):
        table = torch.zeros(2, 8, dtype=torch.int32, device=dev)
        table[1, 0] = entry
        eng.step_paged(ints, ints.clone(), pool, table)
        with pytest.raises(_lib.B2DError) as e:
            eng.check_device()
        assert e.value.status == _lib.B2D_ERR_DEVICE_INPUT
        eng.reset()


def test_switching_a_workspace(engine_tiny):
    """16 to 4 bits and back: the bf16 steps give what they gave before."""
    from transformer_b200.config import CONFIG_TINY as cfg
    eng = DecodeEngine(engine_tiny.w, max_batch=2)
    dev = eng.device
    tok = torch.tensor([3, 5], dtype=torch.int32, device=dev)
    pos, nt = torch.zeros_like(tok), torch.zeros_like(tok)
    table = torch.arange(16, dtype=torch.int32, device=dev).view(2, 8)
    pool, lg = eng.new_kv_pool(16), torch.zeros(2, cfg.vocab_size, device=dev)
    for _ in range(3):
        eng.step_paged(tok, pos, pool, table, lg, nt)
    want = lg.clone()
    _lib.check(eng.lib.b2d_workspace_kv_bits(eng.ws, 4), "kv_bits")
    eng.kv_bits = 4
    pool4 = eng.new_kv_pool(16)
    eng.step_paged(tok, pos, pool4, table, lg, nt)
    _lib.check(eng.lib.b2d_workspace_kv_bits(eng.ws, 16), "kv_bits")
    eng.kv_bits = 16
    lg.zero_()
    eng.step_paged(tok, pos, pool, table, lg, nt)
    assert torch.equal(lg, want)
    eng.check_device()
    eng.close()


@pytest.mark.parametrize("fuse,pipe", [(True, True), (False, False)])
def test_batcher_on_a_4_bit_pool(tiny4, fuse, pipe):
    """Requests through 4 slots and 11 blocks with preemption, as on a bf16
    pool: every request ends with its tokens, every page comes back, and the
    same schedule gives the same tokens."""
    from transformer_b200.config import CONFIG_TINY as cfg

    def serve():
        rng = np.random.default_rng(21)
        cb = ContinuousBatcher(tiny4, 4, 11, admission="optimistic", fuse_prefill=fuse, pipeline=pipe)
        want = {}
        for k in range(10):
            n = int(rng.integers(1, 90))
            g = int(rng.integers(1, cfg.context_len - n + 2))
            kw = dict(temperature=0.7, top_p=0.9, seed=k) if k % 4 == 3 else {}
            want[cb.submit(rng.integers(0, cfg.vocab_size, n), g, **kw)] = g
        got = cb.run()
        tiny4.check_device()
        assert cb.stats["preemptions"] > 0 and cb.pages.n_free == 11
        assert {r: len(t) for r, t in got.items()} == want
        return got

    assert serve() == serve()


# ---- requests with rules ---------------------------------------------------------

def test_rules_of_requests(engine_tiny_batched):
    """Allowed tokens, fixed and by a grammar that ends, biases and penalties,
    next to requests without rules, whose tokens stay what they are alone."""
    from transformer_b200.config import CONFIG_TINY as cfg
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, cfg.vocab_size, n) for n in (5, 20, 33, 7, 12, 9)]

    def batcher():
        return ContinuousBatcher(engine_tiny_batched, 6, 60, pipeline=False)

    plain = batcher()
    alone = [plain.submit(p, 24) for p in prompts]
    alone = [plain.run()[r] for r in alone]

    def grammar(out):  # counts up from 100, then nothing
        return [100 + len(out)] if len(out) < 9 else []

    cb = batcher()
    ids = [cb.submit(prompts[0], 24),
           cb.submit(prompts[1], 24, allowed=np.arange(40, 60), temperature=1.0, top_p=0.95, seed=5),
           cb.submit(prompts[2], 24, allowed=grammar),
           cb.submit(prompts[3], 24, logit_bias={7: 500.0}),
           cb.submit(prompts[4], 24, presence=1000.0),
           cb.submit(prompts[5], 24, frequency=1000.0, temperature=0.5, seed=1)]
    got = cb.run()
    got = [got[i] for i in ids]
    engine_tiny_batched.check_device()
    assert got[0] == alone[0]
    assert len(got[1]) == 24 and all(40 <= t < 60 for t in got[1])
    assert got[2] == list(range(100, 109))
    assert got[3] == [7] * 24
    assert len(set(got[4])) == 24 and len(set(got[5])) == 24
    assert got[4][0] == alone[4][0]
    assert cb.pages.n_free == 60


def test_rules_change_nothing_when_they_say_nothing(engine_tiny_batched):
    """A bias of 0 sends a greedy request through the sampler: the same tokens."""
    from transformer_b200.config import CONFIG_TINY as cfg
    rng = np.random.default_rng(31)
    p = rng.integers(0, cfg.vocab_size, 30)
    out = []
    for kw in ({}, dict(logit_bias={3: 0.0}), dict(allowed=range(cfg.vocab_size))):
        cb = ContinuousBatcher(engine_tiny_batched, 2, 16)
        rid = cb.submit(p, 40, **kw)
        out.append(cb.run()[rid])
    assert out[0] == out[1] == out[2]


def test_a_rule_that_raises_ends_its_request_alone(engine_tiny_batched):
    from transformer_b200.config import CONFIG_TINY as cfg
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, cfg.vocab_size, n) for n in (9, 17, 4)]
    plain = ContinuousBatcher(engine_tiny_batched, 3, 40)
    ids = [plain.submit(p, 20) for p in prompts]
    alone = [plain.run()[i] for i in ids]

    def at_once(out):
        raise KeyError("no rule")

    def later(out):
        return [5] if len(out) < 3 else [cfg.vocab_size]

    cb = ContinuousBatcher(engine_tiny_batched, 3, 40)
    ids = [cb.submit(prompts[0], 20), cb.submit(prompts[1], 20, allowed=at_once),
           cb.submit(prompts[2], 20, allowed=later)]
    got = cb.run()
    assert got[ids[0]] == alone[0] and got[ids[1]] == [] and got[ids[2]] == [5, 5, 5]
    assert set(cb.errors) == set(ids[1:])
    assert isinstance(cb.errors[ids[1]], KeyError) and isinstance(cb.errors[ids[2]], ValueError)
    assert cb.pages.n_free == 40
    again = cb.submit(prompts[1], 20)
    assert cb.run()[again] == alone[1]
