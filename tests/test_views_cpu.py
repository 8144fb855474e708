"""CPU: which views of a buffer share bytes (the operators take an output that
is its input or apart from it), against sets of addresses."""

from __future__ import annotations

import random

import pytest
import torch

from transformer_b200.kv4 import _folded, _overlap, _same_place


def places(x):
    e = x.element_size()
    at = [x.data_ptr()]
    for n, s in zip(x.shape, x.stride()):
        at = [a + i * s * e for a in at for i in range(n)]
    return [a + b for a in at for b in range(e)]


def view(rng, buf, shape, strides=None):
    """A view of these sizes somewhere in buf, contiguous in its last dim."""
    rows, heads, d = shape
    if strides is None:
        strides = rng.choice([(heads * d, d), (heads * d + rng.randint(0, 9), d), (d, rows * d), (d + 1, rows * (d + 1)),
                              (rng.randint(0, 20), rng.randint(0, 20)), (2 * d, d), (3 * heads * d, d),
                              (2 * heads * (d + 1), d + 1)])
    size = (rows - 1) * strides[0] + (heads - 1) * strides[1] + d
    x = torch.as_strided(buf, shape, (*strides, 1), rng.randint(0, buf.numel() - size))
    return x


@pytest.mark.parametrize("seed", range(4))
def test_views_against_their_addresses(seed):
    rng = random.Random(seed)
    half = torch.zeros(600, dtype=torch.float16)
    word = half.view(torch.float32)
    hit = miss = folded = 0
    for _ in range(3000):
        shape = (rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 5))
        x = view(rng, half, shape)
        y = view(rng, rng.choice((half, word)), (*shape[:1], rng.randint(1, 4), shape[2]),
                 rng.choice((None, x.stride()[:2])))
        a, b = places(x), places(y)
        assert _overlap(x, y) == _overlap(y, x) == bool(set(a) & set(b))
        assert _folded(x) == (len(set(a)) < len(a))
        hit, miss, folded = hit + bool(set(a) & set(b)), miss + (not set(a) & set(b)), folded + _folded(x)
    assert min(hit, miss, folded) > 200


def test_empty_and_equal_views():
    buf = torch.zeros(8, 6, 4)
    assert not _overlap(buf[:0], buf) and not _overlap(buf, buf[:, :0]) and not _folded(buf[:0])
    assert not _folded(buf[:, 1:, :2]) and _folded(buf[:1].expand(3, 6, 4))
    assert _same_place(buf, buf.view(8, 6, 4)) and _same_place(buf[:1], buf[0].as_strided((1, 6, 4), (99, 4, 1)))
    assert not _same_place(buf[:, :2], buf.view(16, 3, 4)[:8, :2])


def test_a_pool_off_16_bytes_is_refused():
    """Its pages are copied 16 bytes at a time; a view that starts between is
    refused on the host."""
    import types

    from transformer_b200.config import CONFIG_TINY as cfg
    from transformer_b200.kv4 import page_bytes
    from transformer_b200.multi_sm_decode import DecodeEngine
    eng = types.SimpleNamespace(cfg=cfg, kv_bits=4, device=torch.device("cpu"))
    shape = (cfg.n_layers, 3, cfg.n_kv_heads, page_bytes(cfg.d_head))
    size = 3 * cfg.n_layers * cfg.n_kv_heads * page_bytes(cfg.d_head)
    buf = torch.zeros(size + 64, dtype=torch.uint8)
    base = -buf.data_ptr() % 16
    for off in range(17):
        pool = buf[base + off:base + off + size].view(shape)
        if off % 16:
            with pytest.raises(ValueError):
                DecodeEngine._check_pool(eng, pool)
        else:
            DecodeEngine._check_pool(eng, pool)
