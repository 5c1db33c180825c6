"""What a paged cache refuses at the ends of its ranges, and what its binding refuses of the operands it is handed: no GPU."""

from __future__ import annotations

import ctypes

import pytest
from test_paged import ONE, step


def test_more_heads_behind_a_prefix_than_the_last_launch_counts():
    """Refused before anything is launched, however the prefix would be read."""
    from limn_b200._lib import last_error, lib

    pairs = (ctypes.c_longlong * 4)(256, 64, 256, 64)
    for heads, kv_heads in ((262144, 65536), (1 << 21, 1 << 21)):
        s = step(heads=heads, kv_heads=kv_heads, tokens=1, batch=1)
        assert lib().limn_b200_sdpa_paged_prefix(ctypes.byref(s), ONE, ONE, ONE, pairs, ONE, 30, 1, 0.125, ONE, 1 << 50, None) == 2
        assert "heads" in last_error() and lib().limn_b200_last_launch_count() == 0
    s = step(heads=262140, kv_heads=65535, tokens=0)
    assert lib().limn_b200_sdpa_paged_prefix(ctypes.byref(s), ONE, ONE, ONE, pairs, ONE, 30, 1, 0.125, ONE, 1 << 50, None) == 0
