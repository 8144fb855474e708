"""GPU: requests of the continuous batcher whose rules act together, against the
logits adjustment's definition in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from test_logits_gpu import defined
from transformer_b200.serve import ContinuousBatcher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pipeline", [True, False])
def test_rules_and_repetition_together(engine_tiny_batched, pipeline):
    """Greedy requests with a repetition penalty next to presence, frequency,
    biases and masks: each token has the largest adjusted logit."""
    from transformer_b200.config import CONFIG_TINY as cfg
    rng = np.random.default_rng(17)
    cb = ContinuousBatcher(engine_tiny_batched, 4, 40, pipeline=pipeline)
    rules = {}
    for k in range(8):
        kw = dict(rep_penalty=float(rng.uniform(0.7, 1.6)))
        if k % 2:
            kw.update(presence=float(rng.normal()), frequency=float(rng.normal()))
        if k % 3:
            ids = rng.permutation(cfg.vocab_size)[:20]
            kw["logit_bias"] = {int(t): float(b) for t, b in zip(ids, 3 * rng.normal(size=20))}
        if k % 4 == 2:
            kw["allowed"] = rng.permutation(cfg.vocab_size)[:cfg.vocab_size // 2]
        rules[cb.submit(rng.integers(0, cfg.vocab_size, int(rng.integers(1, 40))), 30, **kw)] = kw
    orig, wrong, seen = cb._sample_rows, [], 0

    def recording(logits, rows, greedy_src):
        nonlocal seen
        rows = list(rows)
        before = logits[:len(rows)].float().cpu().numpy().copy()
        out = orig(logits, rows, greedy_src)
        for lg, r, t in zip(before, rows, out):
            if r is None:
                continue
            kw = rules[r.rid]
            one = np.ones(1, np.float32)
            bias = kw.get("logit_bias", {})
            allowed = np.ones((1, (cfg.vocab_size + 31) // 32 * 32), bool)
            if "allowed" in kw:
                allowed[:] = False
                allowed[0, kw["allowed"]] = True
            x, err = defined(lg[None], np.array([r.out or [0]], np.int32), np.array([len(r.out)]), None,
                             one * np.float32(kw["rep_penalty"]), one * np.float32(kw.get("presence", 0)),
                             one * np.float32(kw.get("frequency", 0)), np.array([list(bias) or [0]], np.int32),
                             np.array([list(bias.values()) or [0.0]], np.float32), np.array([len(bias)]),
                             np.packbits(allowed, axis=1, bitorder="little").view(np.int32))
            seen += 1
            if x[0, t] + err[0, t] < (x[0] - err[0]).max():
                wrong.append((r.rid, len(r.out), int(t), int(x[0].argmax())))
        return out

    cb._sample_rows = recording
    got = cb.run()
    engine_tiny_batched.check_device()
    assert not wrong, wrong[:5]
    assert seen == sum(map(len, got.values())) == 8 * 30


def test_lists_without_room(cuda):
    """A history and biases of no entries (the first step of a batch) change
    nothing; lists that are no matrices are refused."""
    import torch
    from transformer_b200.generate import adjust_logits
    lg = torch.randn(3, 70, device=cuda)
    zero, one = torch.zeros(3, dtype=torch.int32, device=cuda), torch.ones(3, device=cuda)
    none = torch.zeros(3, 0, dtype=torch.int32, device=cuda)
    kw = dict(history=none, hist_len=zero, prompt_len=zero, rep_penalty=2 * one, presence=one, frequency=one)
    assert torch.equal(adjust_logits(lg, **kw), lg)
    bias = dict(bias_ids=none, bias_values=none.float(), bias_len=zero)
    assert torch.equal(adjust_logits(lg, **bias, **kw), lg)
    allowed = torch.full((3, 3), 6, dtype=torch.int32, device=cuda)
    got = adjust_logits(lg, **bias, **kw, allowed=allowed)
    keep = torch.arange(70, device=cuda) % 32
    keep = (keep == 1) | (keep == 2)
    assert torch.equal(got[:, keep], lg[:, keep]) and torch.isneginf(got[:, ~keep]).all()
    for bad in (dict(history=zero[0], hist_len=zero), dict(allowed=zero[0]), dict(history=none, hist_len=zero[:2]),
                dict(bias_ids=none, bias_values=none, bias_len=zero),
                dict(bias_ids=zero, bias_values=one, bias_len=zero)):
        with pytest.raises(ValueError):
            adjust_logits(lg, **bad)
