"""A paged key and value cache on the GPU where its documentation leaves room: idle places of a batch, offsets that fall, scores of any size, kernels that give
up in the middle of a call, what one operator leaves for the next. Against the definitions in float64 (paged_scene.py, which derives the tolerances)."""

from __future__ import annotations

import numpy as np
import pytest
from paged_scene import Scene

pytestmark = pytest.mark.gpu

IDLE = [(0, 0)] * 4000  # so many places that a prefix is read once for the whole batch (sequences without tokens cost nothing, but count)


def launches() -> int:
    from limn_b200._lib import lib

    return lib().limn_b200_last_launch_count()


# ---------------------------------------------------------------- places of a batch that no sequence has

@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("prefix, idle", [(0, []), (0, [(0, 0)] * 500), (700, []), (700, IDLE)], ids=["alone", "alone, more than a block adds up at once", "behind", "behind, read once"])
def test_a_place_that_brings_no_token_may_have_any_length(new, prefix, idle):
    """Its offsets are equal; what its length says, left over from an earlier step or never written, is of no concern and no error."""
    from limn_b200 import runtime

    seqs = [(0, 0), (new, 300), (0, 0), (0, 0), (new, 90), (0, 0)] + idle
    s = Scene(seqs, heads=4, kv_heads=2, hd=64, page_size=16, seed=41, prefix=prefix)
    keys = np.array([*s.keys, 0], np.int64)
    stale = np.array([-1, 2**31 - 1, -(2**31), 16 * s.max_pages + 1])
    none = np.flatnonzero(np.array(s.new) == 0)
    keys[none] = stale[np.arange(len(none)) % 4]
    s.upload(with_new=False, kv_lens=keys)
    k, v = (runtime.upload(np.concatenate([rows[b][len(rows[b]) - n :] for b, n in enumerate(s.new)])) for rows in (s.k, s.v))
    s.step.append(k, v)
    s.check()
    s.check(causal=False)
    assert launches() == (3 if prefix and idle else 2)


# ---------------------------------------------------------------- scores of any size

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("scale", [2.0**-99, 2.0**-6, 1.0, 2.0**10, 2.0**27, 2.0**99], ids=lambda x: f"2^{int(np.log2(x))}")
def test_the_smallest_and_the_largest_scale(scale, new, hd):
    """Queries and keys of whole numbers, whose products are exact in float32, up to 16 * hd, and scales that are powers of two: what is left of the score's error is the
    rounding of log2(e) * scale, 2^-23 of the distance to the row's largest score. A weight that counts is at most 2^-30 of the largest, 21 away: 2^-18, inside the
    comparison's 2^-13. L's 2^-23 of itself is the rounding of the largest score's product with the scale, and of the sum. Tied scores share their row."""
    rng = np.random.default_rng(43)
    s = Scene([(new, 700), (1, 90), (min(new, 5), 2000)], heads=4, kv_heads=2, hd=hd, seed=42)
    s.q = rng.integers(-4, 5, s.q.shape).astype(np.float32).astype(s.dtype)
    s.k = [rng.integers(-4, 5, k.shape).astype(np.float32).astype(s.dtype) for k in s.k]
    s.upload().check(scale=scale)


@pytest.mark.parametrize("idle", [[], IDLE], ids=["for each", "read once"])
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("scale", [2.0**20, 2.0**99], ids=lambda x: f"2^{int(np.log2(x))}")
def test_the_largest_scale_behind_a_prefix(scale, new, idle):
    rng = np.random.default_rng(45)
    s = Scene([(new, 700), (1, 90)] + idle, heads=4, kv_heads=2, hd=64, seed=44, prefix=500)
    s.q = rng.integers(-4, 5, s.q.shape).astype(np.float32).astype(s.dtype)
    s.k = [rng.integers(-4, 5, k.shape).astype(np.float32).astype(s.dtype) for k in s.k]
    s.prefix_k = rng.integers(-4, 5, s.prefix_k.shape).astype(np.float32).astype(s.dtype)
    s.upload().check(scale=scale)
    assert launches() == (3 if idle else 2)
