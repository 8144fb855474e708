"""GPU: the logits adjustment (b2d_adjust_logits) against its definition in
64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from transformer_b200.generate import adjust_logits

pytestmark = pytest.mark.gpu


def defined(logits, hist=None, hist_len=None, prompt_len=None, rep=None, presence=None, frequency=None, bias_ids=None,
            bias_values=None, bias_len=None, allowed=None):
    """(result, allowed error): float64.  Off by a rounding (2^-24 of the
    operands) in each of: the division or product, the penalties' product and
    sum, their subtraction, the bias's addition."""
    x = logits.astype(np.float64)
    err = np.zeros_like(x)
    u = 2.0 ** -24
    b, v = x.shape
    for r in range(b):
        if hist is not None:
            n = min(max(int(hist_len[r]), 0), hist.shape[1])
            made = max(int(prompt_len[r]), 0) if prompt_len is not None else 0
            ids = hist[r, :n]
            for t in np.unique(ids[(ids >= 0) & (ids < v)]):
                if rep is not None:
                    x[r, t] = x[r, t] / float(rep[r]) if x[r, t] > 0 else x[r, t] * float(rep[r])
                    err[r, t] += u * abs(x[r, t])
                c = int((ids[made:] == t).sum())
                if c:
                    take = (float(frequency[r]) if frequency is not None else 0.0) * c + (
                        float(presence[r]) if presence is not None else 0.0)
                    x[r, t] -= take
                    err[r, t] += u * (2 * abs(take) + abs(x[r, t]))
        if bias_ids is not None:
            last = {int(i): float(w) for i, w in zip(bias_ids[r, :max(int(bias_len[r]), 0)],
                                                     bias_values[r, :max(int(bias_len[r]), 0)])}
            for t, w in last.items():
                if 0 <= t < v:
                    x[r, t] += w
                    err[r, t] += u * (abs(x[r, t]) + abs(w))
        if allowed is not None:
            t = np.arange(v)
            x[r, (allowed[r].view(np.uint32)[t // 32] >> (t % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return x, err * 2 + 1e-45


def rules(rng, b, v, cap=40, n_bias=5, density=0.5):
    w = (v + 31) // 32
    return dict(hist=rng.integers(-2, v + 3, (b, cap)).astype(np.int32) % (v + 2) - 1,
                hist_len=rng.integers(0, cap + 1, b).astype(np.int32),
                prompt_len=rng.integers(0, cap + 1, b).astype(np.int32),
                rep=rng.uniform(0.7, 1.6, b).astype(np.float32), presence=rng.normal(size=b).astype(np.float32),
                frequency=rng.normal(size=b).astype(np.float32),
                bias_ids=rng.integers(-1, v + 1, (b, n_bias)).astype(np.int32),
                bias_values=rng.normal(size=(b, n_bias)).astype(np.float32),
                bias_len=rng.integers(0, n_bias + 1, b).astype(np.int32),
                allowed=np.packbits(rng.random((b, w * 32)) < density, axis=1, bitorder="little").view(np.int32))


NAMES = {"hist": "history", "rep": "rep_penalty"}


def call(logits, kw, cuda, out=None):
    dev = {NAMES.get(n, n): torch.from_numpy(np.ascontiguousarray(a)).to(cuda) for n, a in kw.items()}
    return adjust_logits(logits, out=out, **dev)


def compare(got, want, err):
    g = got.double().cpu().numpy()
    assert np.array_equal(np.isneginf(g), np.isneginf(want))
    f = np.isfinite(want)
    assert (np.abs(g - want)[f] <= err[f]).all()


@pytest.mark.parametrize("b,v", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 1000), (2, 4096), (3, 4097), (7, 32000),
                                 (300, 515), (2, 100003), (80, 40000)])
def test_all_rules(cuda, b, v):
    rng = np.random.default_rng(b * 7 + v)
    lg = (3 * rng.normal(size=(b, v))).astype(np.float32)
    kw = rules(rng, b, v)
    compare(call(torch.from_numpy(lg).to(cuda), kw, cuda), *defined(lg, **kw))


@pytest.mark.parametrize("keep", [["hist", "hist_len", "rep"], ["hist", "hist_len", "prompt_len", "frequency"],
                                  ["hist", "hist_len", "presence"], ["hist", "hist_len"],
                                  ["bias_ids", "bias_values", "bias_len"], ["allowed"], []])
def test_single_rules(cuda, keep):
    rng = np.random.default_rng(len(keep))
    lg = rng.normal(size=(4, 5000)).astype(np.float32)
    kw = {n: a for n, a in rules(rng, 4, 5000).items() if n in keep}
    compare(call(torch.from_numpy(lg).to(cuda), kw, cuda), *defined(lg, **kw))


def test_repeats_and_long_lists(cuda):
    """One token thousands of times, an id biased many times (the last counts),
    lists longer than the vocabulary, and the same bits from every run."""
    rng = np.random.default_rng(3)
    b, v, cap = 3, 37, 6000
    lg = rng.normal(size=(b, v)).astype(np.float32)
    kw = rules(rng, b, v, cap, 900, 1.0)
    kw["hist"][0] = 5
    kw["hist_len"][:] = [cap, cap + 100, -4]
    kw["prompt_len"][:] = [1000, -3, 0]
    kw["bias_len"][:] = 900
    lg_d = torch.from_numpy(lg).to(cuda)
    got = call(lg_d, kw, cuda)
    compare(got, *defined(lg, **kw))
    for _ in range(3):
        assert torch.equal(call(lg_d, kw, cuda), got)


def test_nothing_allowed_and_infinite_logits(cuda):
    lg = np.array([[np.inf, -np.inf, 1.0, -2.0] * 10] * 2, np.float32)
    kw = dict(allowed=np.array([[0, 0], [-1, -1]], np.int32), hist=np.array([[0, 1], [0, 1]], np.int32),
              hist_len=np.array([2, 2], np.int32), rep=np.array([2, 2], np.float32))
    got = call(torch.from_numpy(lg).to(cuda), kw, cuda).cpu().numpy()
    assert np.isneginf(got[0]).all() and np.array_equal(got[1], lg[1])


def test_in_place_strided_and_streamed(cuda):
    """Rows of a wider buffer, `out` the logits themselves, another stream, a
    captured call replayed on new logits."""
    rng = np.random.default_rng(8)
    b, v = 6, 2049
    kw = rules(rng, b, v)
    lg = rng.normal(size=(b, v)).astype(np.float32)
    want = call(torch.from_numpy(lg).to(cuda), kw, cuda)
    wide = torch.full((b, v + 31), 9.0, device=cuda)
    view = wide[:, 3:3 + v]
    view.copy_(torch.from_numpy(lg))
    assert call(view, kw, cuda, out=view).data_ptr() == view.data_ptr()
    assert torch.equal(view, want) and (wide[:, :3] == 9).all() and (wide[:, 3 + v:] == 9).all()
    dev = {NAMES.get(n, n): torch.from_numpy(a).to(cuda) for n, a in kw.items()}
    buf, out = torch.from_numpy(lg).to(cuda), torch.zeros(b, v, device=cuda)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(cuda)
    adjust_logits(buf, out=out, stream=side, **dev)
    side.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        adjust_logits(buf, out=out, **dev)
    buf.mul_(-0.5)
    g.replay()
    assert torch.equal(out, adjust_logits(buf, **dev))


def test_refusals(cuda):
    lg = torch.zeros(2, 64, device=cuda)
    ints = torch.zeros(2, 3, dtype=torch.int32, device=cuda)
    one = torch.zeros(2, dtype=torch.int32, device=cuda)
    for kw in (dict(history=ints), dict(hist_len=one), dict(rep_penalty=torch.ones(2, device=cuda)),
               dict(history=ints, hist_len=one[:1]), dict(history=ints.long(), hist_len=one),
               dict(bias_ids=ints, bias_len=one), dict(allowed=ints[:, :1].contiguous()), dict(allowed=ints.T),
               dict(history=ints, hist_len=one, presence=torch.ones(2, device=cuda).double()),
               dict(out=torch.zeros(2, 63, device=cuda)), dict(history=ints.cpu(), hist_len=one)):
        with pytest.raises(ValueError):
            adjust_logits(lg, **kw)
    with pytest.raises(ValueError):
        adjust_logits(lg.half())
    with pytest.raises(ValueError):
        adjust_logits(lg.T)
