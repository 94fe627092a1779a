"""Sizes past which the 4-bit cache's calls refuse (before any device is touched)."""
from __future__ import annotations

import ctypes as C

import pytest

from chatnet_b200 import _native as N
from tests.test_kvq4 import _CTX, _P, INVALID, _append, _attend, _cache


def _read(cache):
    return N.lib().cn_kvq4_read_dev(_CTX, C.byref(cache), _P, _P, 128, _P, 0, 1, 1, None)


@pytest.mark.parametrize("ctx_len", [(1 << 30) + 8, (1 << 31) - 8])
def test_more_positions_than_a_tile_can_be_rounded_up_from(ctx_len):
    cache = _cache(ctx_len=ctx_len)
    assert _append(cache) == INVALID and _attend(cache) == INVALID and _read(cache) == INVALID
    assert str(ctx_len) in N.last_error()
