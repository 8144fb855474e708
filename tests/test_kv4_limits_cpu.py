"""CPU: limits of the attention call's numbers (refused on the host)."""

from __future__ import annotations

import ctypes

import pytest

from test_kv4_cpu import BAD, cache, query
from transformer_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from transformer_b200 import build
    build.build()
    return _lib.load()


@pytest.mark.parametrize("scale", [3.4e38, 2.5e38])
def test_scales_that_overflow_are_refused(lib, scale):
    """The kernels scale by log2(e) more, which has to stay finite."""
    n = ctypes.c_uint64(7)
    c, q = cache(), query(scale=scale)
    assert lib.b2d_kv4_attention_scratch(ctypes.byref(c), ctypes.byref(q), ctypes.byref(n)) == BAD and n.value == 0
    assert lib.b2d_kv4_attention(ctypes.byref(c), ctypes.byref(q), None, 0, None) == BAD
