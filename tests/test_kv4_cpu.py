"""CPU: the refusals of the 4-bit cache's and the logits adjustment's entry
points (no GPU work: every call is refused on the host), and the test
definitions' own consistency."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kv4_ref as R
from transformer_b200 import _lib

P = 0x100000  # an address that is never dereferenced


@pytest.fixture(scope="module")
def lib():
    from transformer_b200 import build
    build.build()
    return _lib.load()


def cache(**kw):
    f = dict(pool=P, table=P, status=None, n_kv_heads=4, d_head=64, num_blocks=8, blocks_per_seq=4, table_rows=2,
             device=0)
    f.update(kw)
    return _lib.Kv4Cache(**f)


def rows(**kw):
    f = dict(q=P, k=P, v=P, q_out=P + 4096, q_row=2048, q_head=64, k_row=512, k_head=64, v_row=512, v_head=64,
             q_out_row=1024, q_out_head=64, pos=P, seq=P, cos=P, sin=P, dtype=_lib.B2D_BF16, q_out_dtype=_lib.B2D_BF16,
             n_rows=3, n_heads=16, rotary_dim=64, interleaved=0, max_pos=64)
    f.update(kw)
    return _lib.Kv4Rows(**f)


def query(**kw):
    f = dict(q=P, out=P, q_row=1024, q_head=64, out_row=1024, out_head=64, lens=P, q_start=None, dtype=_lib.B2D_BF16,
             n_rows=2, n_heads=16, n_seqs=2, max_rows=1, max_len=64, scale=0.125)
    f.update(kw)
    return _lib.Kv4Query(**f)


BAD, NO = _lib.B2D_ERR_INVALID_ARG, _lib.B2D_ERR_UNSUPPORTED
BAD_CACHE = [(dict(pool=None), BAD), (dict(pool=P + 8), BAD), (dict(table=None), BAD), (dict(n_kv_heads=0), BAD),
             (dict(num_blocks=0), BAD), (dict(blocks_per_seq=0), BAD), (dict(table_rows=0), BAD), (dict(device=-1), BAD),
             (dict(blocks_per_seq=1 << 28), BAD), (dict(d_head=32), NO), (dict(d_head=96), NO), (dict(d_head=256), NO)]


@pytest.mark.parametrize("kw,status", BAD_CACHE)
def test_cache_refused(lib, kw, status):
    c, n = cache(**kw), ctypes.c_uint64()
    assert lib.b2d_kv4_append(ctypes.byref(c), ctypes.byref(rows()), None) == status
    assert lib.b2d_kv4_read(ctypes.byref(c), P, P, 2, _lib.B2D_BF16, P, P, None) == status
    assert lib.b2d_kv4_attention_scratch(ctypes.byref(c), ctypes.byref(query()), ctypes.byref(n)) == status
    assert lib.b2d_kv4_attention(ctypes.byref(c), ctypes.byref(query()), None, 0, None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(k=None), BAD), (dict(v=None), BAD), (dict(pos=None), BAD), (dict(n_rows=-1), BAD), (dict(q_out=None), BAD),
    (dict(q=None), BAD), (dict(n_heads=0), BAD), (dict(cos=None), BAD), (dict(sin=None), BAD), (dict(rotary_dim=0), BAD),
    (dict(rotary_dim=66), BAD), (dict(rotary_dim=7), BAD), (dict(max_pos=0), BAD), (dict(seq=None), BAD),
    (dict(q_out=P), BAD), (dict(dtype=3), NO), (dict(dtype=-1), NO), (dict(q_out_dtype=_lib.B2D_F16), NO)])
def test_rows_refused(lib, kw, status):
    assert lib.b2d_kv4_append(ctypes.byref(cache()), ctypes.byref(rows(**kw)), None) == status


@pytest.mark.parametrize("args,status", [
    ((None, P, 2, 1, P, P), BAD), ((P, P, -1, 1, P, P), BAD), ((P, None, 3, 1, P, P), BAD), ((P, P, 2, 1, None, P), BAD),
    ((P, P, 2, 1, P, None), BAD), ((P, P, 2, 5, P, P), NO)])
def test_read_refused(lib, args, status):
    assert lib.b2d_kv4_read(ctypes.byref(cache()), *args, None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), BAD), (dict(out=None), BAD), (dict(lens=None), BAD), (dict(n_rows=-1), BAD), (dict(n_rows=3), BAD),
    (dict(n_seqs=-1), BAD), (dict(n_heads=0), BAD), (dict(n_heads=6), BAD), (dict(max_rows=0), BAD),
    (dict(max_rows=2), BAD), (dict(n_seqs=3, n_rows=3), BAD), (dict(max_len=-1), BAD), (dict(max_len=65), BAD),
    (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD), (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD),
    (dict(dtype=_lib.B2D_F32), NO)])
def test_query_refused(lib, kw, status):
    n = ctypes.c_uint64(7)
    assert lib.b2d_kv4_attention_scratch(ctypes.byref(cache()), ctypes.byref(query(**kw)), ctypes.byref(n)) == status
    assert n.value == 0
    assert lib.b2d_kv4_attention(ctypes.byref(cache()), ctypes.byref(query(**kw)), None, 0, None) == status


def rules(**kw):
    f = dict(logits=P, out=P, logits_ld=100, out_ld=100, history=P, hist_len=P, prompt_len=P, rep=P, presence=P,
             frequency=P, bias_ids=P, bias_values=P, bias_len=P, allowed=P, allowed_ld=4, batch=2, vocab=100, hist_cap=8,
             bias_cap=3, device=0)
    f.update(kw)
    return _lib.LogitsRules(**f)


@pytest.mark.parametrize("kw,status", [
    (dict(logits=None), BAD), (dict(out=None), BAD), (dict(batch=-1), BAD), (dict(vocab=0), BAD),
    (dict(logits_ld=99), BAD), (dict(out_ld=99), BAD), (dict(out_ld=101), BAD), (dict(history=None), BAD),
    (dict(hist_len=None), BAD), (dict(hist_cap=-1), BAD), (dict(bias_ids=None), BAD), (dict(bias_values=None), BAD),
    (dict(bias_len=None), BAD), (dict(bias_cap=-1), BAD), (dict(allowed_ld=3), BAD), (dict(device=-1), BAD),
    (dict(batch=70000), NO)])
def test_logits_rules_refused(lib, kw, status):
    assert lib.b2d_adjust_logits(ctypes.byref(rules(**kw)), None) == status


def test_null_structs_refused(lib):
    assert lib.b2d_kv4_append(None, None, None) == BAD
    assert lib.b2d_kv4_append(ctypes.byref(cache()), None, None) == BAD
    assert lib.b2d_kv4_attention(ctypes.byref(cache()), None, None, 0, None) == BAD
    assert lib.b2d_kv4_attention_scratch(ctypes.byref(cache()), ctypes.byref(query()), None) == BAD
    assert lib.b2d_adjust_logits(None, None) == BAD


def test_empty_calls_do_nothing(lib):
    assert lib.b2d_adjust_logits(ctypes.byref(rules(batch=0)), None) == _lib.B2D_OK


def test_python_refusals_on_the_host():
    """Host tensors and wrong shapes are refused before the library is asked."""
    from transformer_b200.generate import adjust_logits
    from transformer_b200.kv4 import kv4_append, kv4_attention, kv4_read, new_kv4_pool
    pool = new_kv4_pool(2, 1, 64, "cpu")
    ints = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 1, dtype=torch.int32)
    k = torch.zeros(2, 1, 64)
    for call in (lambda: kv4_append(pool, k, k, ints, table), lambda: kv4_read(pool, ints, table),
                 lambda: kv4_attention(k.half(), pool, ints, table), lambda: adjust_logits(torch.zeros(2, 8)),
                 lambda: new_kv4_pool(2, 1, 96, "cpu"), lambda: new_kv4_pool(0, 1, 64, "cpu")):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("d", [64, 128])
def test_layout_is_a_permutation(d):
    """Every nibble and scale byte of a page belongs to one slot and dim."""
    nib, scale = set(), {}
    for where in (R.k_bytes, R.v_bytes):
        for r in range(16):
            for i in range(d):
                b, hi, s = where(d, r, i)
                nib.add((b, hi))
                scale.setdefault((where.__name__, r, i // 16), set()).add(s)
    assert len(nib) == 2 * 16 * d
    assert all(len(s) == 1 for s in scale.values()) and len(set().union(*scale.values())) == 2 * d
    assert not {b for b, _ in nib} & set().union(*scale.values())
    assert {b for b, _ in nib} | set().union(*scale.values()) == set(range(18 * d))


def test_held_values_are_exact_in_16_bits():
    rng = np.random.default_rng(0)
    x = rng.normal(size=(4000, 64)) * np.exp(rng.normal(size=(4000, 1)) * 6)
    h = R.held(x)
    for t in (torch.bfloat16, torch.float16):
        assert np.array_equal(torch.from_numpy(h).to(t).double().numpy(), h)
    inside = np.abs(x) <= 64512
    s = np.abs(x.reshape(4000, 4, 16)).max(-1, keepdims=True)
    # a code is at most half a scale off; the scale is at most 8/7 of amax / 7 (or 2^-17 above it)
    off = np.abs(h - x).reshape(4000, 4, 16)
    assert (off <= s / 7 * (9 / 8) / 2 + 2.0 ** -18)[inside.reshape(off.shape)].all()


def test_held_on_ties_goes_to_even():
    g = np.array([7, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 6.5] + [0] * 8, np.float64)
    assert list(R.held(g)[:8]) == [7, 0, 2, 2, 0, -2, -2, 6]


def test_submit_refuses_bad_rules():
    from test_serve_cpu import FakeEngine
    from transformer_b200.serve import ContinuousBatcher
    cb = ContinuousBatcher(FakeEngine(), 4, 16)
    for kw in (dict(presence=float("nan")), dict(frequency=float("inf")), dict(logit_bias={97: 1.0}),
               dict(logit_bias={-1: 1.0}), dict(logit_bias={3: float("nan")}), dict(allowed=[]), dict(allowed=[97]),
               dict(allowed=[-1])):
        with pytest.raises(ValueError):
            cb.submit([1, 2], 4, **kw)
    assert cb.idle()
    rid = cb.submit([1, 2], 4, presence=0.0, frequency=0.0, logit_bias={})
    assert not cb.waiting[0].rules and cb.waiting[0].greedy and rid == 0


def test_workspace_kv_bits_refused(lib):
    assert lib.b2d_workspace_kv_bits(None, 4) == BAD
