"""CPU: rules that requests of the continuous batcher bring, on the host: their
order, and what submit refuses."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_serve_cpu import FakeEngine
from transformer_b200.serve import ContinuousBatcher

VOCAB = 97


class PlainSampler:
    """Penalises and takes the largest logit, as the device's does at temperature 0."""

    def __init__(self, rows, cap):
        self.history, self.hist_len = torch.zeros(rows, cap, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
        self.uniforms = torch.zeros(rows, dtype=torch.float64)

    def sample(self, logits, temperature, top_p, rep_penalty, m):
        x = logits[:m].double().numpy().copy()
        for i in range(m):
            seen = np.unique(self.history[i, :int(self.hist_len[i])].numpy())
            x[i, seen] = np.where(x[i, seen] > 0, x[i, seen] / rep_penalty, x[i, seen] * rep_penalty)
        return torch.from_numpy(x.argmax(-1).astype(np.int32))


def plain_adjust(logits, *, out, history, hist_len, presence, frequency, rep_penalty=None, bias_ids=None,
                 bias_values=None, bias_len=None, allowed=None):
    """adjust_logits by its definition, in place."""
    assert out.data_ptr() == logits.data_ptr()
    for i in range(logits.shape[0]):
        x = logits[i].double().numpy().copy()
        ids, count = np.unique(history[i, :int(hist_len[i])].numpy(), return_counts=True)
        if rep_penalty is not None:
            rp = float(rep_penalty[i])
            x[ids] = np.where(x[ids] > 0, x[ids] / rp, x[ids] * rp)
        x[ids] -= float(frequency[i]) * count + float(presence[i])
        if bias_ids is not None:
            for t, b in zip(bias_ids[i, :int(bias_len[i])].tolist(), bias_values[i].tolist()):
                x[t] += b
        if allowed is not None:
            words = allowed[i].numpy().view(np.uint32)
            t = np.arange(VOCAB)
            x[(words[t // 32] >> (t % 32).astype(np.uint32)) & 1 == 0] = -np.inf
        logits[i] = torch.from_numpy(x)
    return out


def batcher(monkeypatch):
    import transformer_b200.generate as G
    monkeypatch.setattr(G, "adjust_logits", plain_adjust)
    cb = ContinuousBatcher(FakeEngine(vocab=VOCAB), 4, 16)
    cb._sampler = PlainSampler(4, cb._hist_cap)
    return cb


def test_repetition_comes_before_the_other_rules(monkeypatch):
    """Logit 2, seen: 2 / 1.3 - 4 = -2.46 beats -2.55, and (2 - 4) 1.3 = -2.6 does
    not; the same with penalties in the bias's place."""
    for kw in (dict(logit_bias={5: -4.0}), dict(presence=4.0), dict(frequency=2.0)):
        cb = batcher(monkeypatch)
        cb.submit([1], 8, rep_penalty=1.3, **kw)
        r = cb.waiting[0]
        r.out = [5, 5]
        lg = torch.full((1, VOCAB), -50.0)
        lg[0, 5], lg[0, 6] = 2.0, -2.55
        assert cb._sample_rows(lg, [r], torch.zeros(1, dtype=torch.int32)).tolist() == [5]


def test_rows_with_and_without_rules(monkeypatch):
    """A batch of all kinds, each row's token by the definition in its order."""
    rng = np.random.default_rng(0)
    for _ in range(30):
        cb = batcher(monkeypatch)
        kinds = [dict(), dict(rep_penalty=1.7), dict(rep_penalty=1.4, presence=0.7, frequency=-0.3,
                                                     logit_bias={t: (-1.5, 0.75)[t % 2] for t in range(VOCAB)}),
                 dict(rep_penalty=0.6, allowed=rng.permutation(VOCAB)[:20])]
        for kw in kinds:
            cb.submit([1, 2], 40, **kw)
        rows, lg = list(cb.waiting), rng.normal(size=(4, VOCAB)).astype(np.float32)
        want = []
        for r, kw, x in zip(rows, kinds, lg.astype(np.float64)):
            r.out = rng.choice(np.argsort(-x)[:8], int(rng.integers(0, 30))).tolist()
            for t in set(r.out):
                rp = float(np.float32(r.rep_penalty))
                x[t] = x[t] / rp if x[t] > 0 else x[t] * rp
                x[t] -= kw.get("frequency", 0.0) * r.out.count(t) + kw.get("presence", 0.0)
            for t, b in kw.get("logit_bias", {}).items():
                x[t] += b
            if "allowed" in kw:
                x[np.setdiff1d(np.arange(VOCAB), kw["allowed"])] = -np.inf
            want.append(int(x.argmax()))
        argmax = torch.from_numpy(lg.argmax(-1).astype(np.int32))
        assert cb._sample_rows(torch.from_numpy(lg), rows, argmax).tolist() == want


@pytest.mark.parametrize("kw", [dict(presence=1e300), dict(frequency=-1e39), dict(logit_bias={1: 0.5, 3: 3.5e38}),
                                dict(logit_bias={0: -1e200}), dict(presence=2.0 ** 128)])
def test_numbers_that_float32_does_not_hold_are_refused(kw):
    """They would be infinite where they act."""
    cb = ContinuousBatcher(FakeEngine(vocab=VOCAB), 4, 16)
    with pytest.raises(ValueError):
        cb.submit([1], 4, **kw)
    assert cb.idle()
    top = float(np.finfo(np.float32).max)
    cb.submit([1], 4, presence=top, frequency=-top, logit_bias={3: top, 4: -top, 5: 1e-300})


@pytest.mark.parametrize("ids", [np.arange(VOCAB) % 2 == 0, [True, False], [1.0, 2.0], np.array([3.5]), ["5"],
                                 np.array([2 ** 63 + 4], np.uint64), [None]])
def test_allowed_takes_token_ids_only(monkeypatch, ids):
    """A mask of the vocabulary (or other things that are no ids) is refused, and
    ends its request when a function gives it."""
    cb = batcher(monkeypatch)
    with pytest.raises(ValueError):
        cb.submit([1], 4, allowed=ids)
    assert cb.idle()
    rid = cb.submit([1], 4, allowed=lambda out: ids)
    assert cb._sample_rows(torch.zeros(1, VOCAB), [cb.waiting[0]], torch.zeros(1, dtype=torch.int32)).tolist() == [-1]
    assert isinstance(cb.errors[rid], ValueError)


def test_allowed_is_kept_as_it_was_given(monkeypatch):
    cb = batcher(monkeypatch)
    for ids in ({5, 7}, range(3), np.array([[9, 11]], np.uint8), [np.int32(4)], np.array([8], np.uint64)):
        cb.submit([1], 4, allowed=ids)
    mine = np.array([20, 30])
    cb.submit([1], 4, allowed=mine)
    mine[:] = VOCAB
    got = [sorted(r.allowed.tolist()) for r in cb.waiting]
    assert got == [[5, 7], [0, 1, 2], [9, 11], [4], [8], [20, 30]]
    cb.submit([1], 4, allowed=lambda out: [])
    assert cb._sample_rows(torch.zeros(1, VOCAB), [cb.waiting[-1]], torch.zeros(1, dtype=torch.int32)).tolist() == [-1]
    assert not cb.errors


@pytest.mark.parametrize("bias", [{3.7: 1.0}, {"5": 1.0}, {True: 1.0}, {np.float32(2): 1.0}, {None: 0.0}])
def test_biases_take_token_ids_only(bias):
    cb = ContinuousBatcher(FakeEngine(vocab=VOCAB), 4, 16)
    with pytest.raises(ValueError):
        cb.submit([1], 4, logit_bias=bias)
    cb.submit([1], 4, logit_bias={np.int32(3): 1, 4: np.float32(0.5)})
    assert cb.waiting[0].logit_bias == {3: 1.0, 4: 0.5} and len(cb.waiting) == 1
