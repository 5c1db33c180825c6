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
