"""A paged key and value cache on the GPU: append, attention over the pages, attention behind a shared prefix, against the definitions
in float64 (paged_scene.py, which derives the tolerances)."""

from __future__ import annotations

import numpy as np
import pytest
from paged_scene import BF16, F16, HALF_STEP, NAMES, NOWHERE, Scene, poison

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- append

APPEND = [
    # dtype, heads, kv_heads, hd, hd_v, rotated, pairing, page size, order, first position, sequences
    (BF16, 4, 2, 64, 64, 64, "halves", 16, "token", 0, [(1, 1)]),
    (BF16, 32, 8, 128, 128, 128, "halves", 16, "token", 0, [(1, 2000), (3, 40), (0, 12), (16, 16)]),
    (F16, 12, 12, 80, 80, 32, "neighbours", 48, "head", 7, [(1, 49), (5, 48), (2, 97)]),
    (BF16, 6, 2, 72, 40, 72, "halves", 8, "token", 1000003, [(9, 9), (1, 8), (7, 70)]),  # a half of 36 columns: 8 bytes at a time
    (F16, 5, 5, 96, 128, 8, "halves", 24, "head", 0, [(30, 31)]),
    (BF16, 7, 1, 8, 8, 8, "neighbours", 8, "token", 3, [(2, 9)] * 70),  # more sequences than a warp probes at once
    (F16, 2, 1, 16, 24, 0, "halves", 256, "token", 0, [(200, 300)]),
    (BF16, 1, 1, 128, 8, 64, "neighbours", 64, "head", 0, [(1, 1)] * 1100),
]


def _turned(x, positions, frequencies, rotated, pairing):
    """x (n, heads, width) in float64, its first columns turned; and how much the operands of each result weigh."""
    x = x.astype(np.float64)
    out, size = x.copy(), np.zeros_like(x)
    if rotated:
        angle = positions[:, None].astype(np.float64) * frequencies
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        a = slice(0, rotated // 2) if pairing == "halves" else slice(0, rotated, 2)
        b = slice(rotated // 2, rotated) if pairing == "halves" else slice(1, rotated, 2)
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
        size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return out, size


@pytest.mark.parametrize("case", APPEND, ids=[f"{NAMES[c[0]]}-{c[3]}x{c[4]}-rot{c[5]}-{c[6]}-page{c[7]}-{c[8]}-{len(c[10])}seq" for c in APPEND])
@pytest.mark.parametrize("queries", ["apart", "in place", "none"])
def test_append(case, queries):
    from limn_b200 import runtime

    dtype, heads, kv_heads, hd, hd_v, rotated, pairing, page_size, order, first, seqs = case
    s = Scene(seqs, dtype=dtype, heads=heads, kv_heads=kv_heads, hd=hd, hd_v=hd_v, page_size=page_size, order=order, spare_tokens=3, seed=5)
    s.upload(with_new=False, first_position=first)
    frequencies = 10000.0 ** (-np.arange(rotated // 2) / max(1, rotated // 2))
    rng = np.random.default_rng(9)
    width = heads * hd + kv_heads * (hd + hd_v)  # q, k and v are slices of one projection
    projected = rng.standard_normal((s.tokens, width)).astype(np.float32).astype(dtype)
    dev, freqs = runtime.upload(projected), runtime.upload(frequencies) if rotated else None
    apart = runtime.upload(poison(dtype, (s.tokens, heads, hd)))
    k_at, v_at = dev.ptr + 2 * heads * hd, dev.ptr + 2 * (heads + kv_heads) * hd
    q = {"apart": {"q": dev, "q_out": apart, "q_strides": (width, hd)}, "none": {},
         "in place": {"q": dev, "q_out": dev, "q_strides": (width, hd), "q_out_strides": (width, hd)}}[queries]
    s.step.append(k_at, v_at, k_strides=(width, hd), v_strides=(width, hd_v), frequencies=freqs, rotated=rotated, pairing=pairing, **q)
    runtime.synchronize()
    assert s.error_bits() == 0

    rows = int(s.start[-1])
    positions = np.concatenate([np.arange(n) + k - n for n, k in seqs]).astype(np.int64) + first
    # a turned value: two products and a sum in float32 of a cosine and a sine that are off by 2 pi 2^-25 (the turn's fraction)
    # and two steps of sincospif: 2^-21 of |x| + |y|, then one rounding
    half = HALF_STEP[dtype]

    def close(have, want, size):
        bound = half * np.abs(want) + 2.0**-21 * (1 + half) * size + (2.0**-25 if dtype == F16 else 0) * (size > 0)
        off = np.abs(have.astype(np.float64) - want)
        assert (off <= bound).all(), f"off by {off.max():.3e}"

    part = projected.astype(np.float64)[:rows]
    want_q, size_q = _turned(part[:, : heads * hd].reshape(rows, heads, hd), positions, frequencies, rotated, pairing)
    want_k, size_k = _turned(part[:, heads * hd : (heads + kv_heads) * hd].reshape(rows, kv_heads, hd), positions, frequencies, rotated, pairing)
    if queries == "apart":
        have = runtime.download(apart, np.uint16, (s.tokens, heads, hd)).view(dtype)
        assert (have[rows:].view(np.uint16) == 0x7FFF).all()
        close(have[:rows], want_q, size_q)
    after = runtime.download(dev, np.uint16, (s.tokens, width)).view(dtype)
    if queries == "in place":
        close(after[:rows, : heads * hd].reshape(rows, heads, hd), want_q, size_q)
        assert np.array_equal(after[rows:].view(np.uint16), projected[rows:].view(np.uint16))
    else:
        assert np.array_equal(after.view(np.uint16), projected.view(np.uint16))
    # the cache: new slots as they should be, everything else bit for bit as it was
    before_k, before_v = s.filled(with_new=False)
    have_k = s.by_slot(runtime.download(s.k_dev, np.uint16, before_k.shape))
    have_v = s.by_slot(runtime.download(s.v_dev, np.uint16, before_v.shape))
    left_k, left_v = s.by_slot(before_k.view(np.uint16)).copy(), s.by_slot(before_v.view(np.uint16)).copy()
    token = 0
    for b, (n, length) in enumerate(seqs):
        for slot in range(length - n, length):
            at = (s.table[b, slot // page_size], slot % page_size)
            close(have_k[at].copy().view(dtype), want_k[token], size_k[token])
            left_k[at] = have_k[at]
            left_v[at] = projected[token, (heads + kv_heads) * hd :].reshape(kv_heads, hd_v).view(np.uint16)
            token += 1
    assert np.array_equal(have_k, left_k) and np.array_equal(have_v, left_v)


# ---------------------------------------------------------------- attention

GENERATION = [(1, 1), (1, 17), (0, 30), (1, 64), (1, 65), (1, 200), (0, 0), (1, 1000), (1, 15), (1, 16)]
DRAFTS = [(4, 4), (1, 63), (3, 64), (2, 129), (4, 500), (0, 9), (2, 2)]
PROMPTS = [(130, 130), (1, 300), (70, 257), (0, 5), (256, 256), (300, 900), (33, 33)]
SHAPES = [
    # id, dtype, heads, kv_heads, hd, hd_v, page size, order, sequences
    ("generation gqa4 128", BF16, 8, 2, 128, 128, 16, "token", GENERATION),
    ("generation mha 64", F16, 3, 3, 64, 64, 64, "head", GENERATION),
    ("generation gqa16 80", F16, 16, 1, 80, 80, 48, "token", GENERATION),
    ("generation 7 to 1, 32", BF16, 7, 1, 32, 32, 8, "token", GENERATION),
    ("generation 128 to 1", BF16, 128, 1, 64, 64, 32, "head", GENERATION[:6]),
    ("generation hd 128 hd_v 64", BF16, 4, 2, 128, 64, 24, "token", GENERATION),
    ("generation hd 64 hd_v 128", F16, 4, 2, 64, 128, 256, "head", GENERATION),
    ("generation hd 8 hd_v 16", BF16, 4, 4, 8, 16, 16, "token", GENERATION),
    ("drafts gqa2 128", BF16, 4, 2, 128, 128, 16, "token", DRAFTS),
    ("drafts gqa5 96", F16, 10, 2, 96, 96, 40, "head", DRAFTS),
    ("drafts gqa8 64", BF16, 8, 1, 64, 64, 16, "token", DRAFTS),
    ("prompts mha 64", BF16, 2, 2, 64, 64, 16, "token", PROMPTS),
    ("prompts gqa4 128", BF16, 8, 2, 128, 128, 64, "head", PROMPTS),
    ("prompts gqa3 80", F16, 6, 2, 80, 80, 48, "token", PROMPTS),
    ("prompts 128 hd_v 48", F16, 4, 2, 128, 48, 128, "token", PROMPTS),
    ("prompts 100 to 1", BF16, 100, 1, 64, 64, 8, "head", [(5, 5), (20, 400), (1, 33)]),
    ("prompts 11 to 1, pages of 256", F16, 11, 1, 128, 128, 256, "token", [(50, 300), (100, 700)]),
]


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("prefix", [0, 5, 300], ids=["alone", "prefix5", "prefix300"])
@pytest.mark.parametrize("shape", SHAPES, ids=[s[0] for s in SHAPES])
def test_attention(shape, prefix, causal):
    _, dtype, heads, kv_heads, hd, hd_v, page_size, order, seqs = shape
    s = Scene(seqs, dtype=dtype, heads=heads, kv_heads=kv_heads, hd=hd, hd_v=hd_v, page_size=page_size, order=order, prefix=prefix, spare_tokens=2,
              seed=11, row_room=8).upload()
    s.check(causal=causal)


@pytest.mark.parametrize("length", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1023, 1025])
@pytest.mark.parametrize("new", [1, 2, 40])
def test_every_length(length, new):
    Scene([(min(new, length), length)], heads=4, kv_heads=1, hd=64, page_size=8, seed=length).upload().check()


@pytest.mark.parametrize("heads", [1, 2, 4])
def test_more_tokens_than_keys(heads):
    """Tokens in front of a sequence's first key see nothing, and with a prefix only that."""
    seqs = [(5, 3), (1, 0), (40, 2), (2, 200)]
    blind = Scene(seqs, heads=heads, kv_heads=1, hd=64, seed=2).upload()
    _, lse = blind.check()
    assert np.isinf(lse[[0, 1, 5]]).all()
    Scene(seqs, heads=heads, kv_heads=1, hd=64, seed=2, prefix=70).upload().check()
    Scene(seqs, heads=heads, kv_heads=1, hd=64, seed=2).upload().check(causal=False)


@pytest.mark.parametrize("mul", [0.0, 1e-3, 8.0])
@pytest.mark.parametrize("new", [1, 100])
def test_flat_and_sharp_weights(mul, new):
    """Scores up to 8 * 30 / 8: the maximum moves again and again; and queries of nothing, the mean of v. (The tolerance of
    a score grows with it: eight times the bound on sum |q k| scale makes 2^-10 of A; the comparison here allows for it.)"""
    s = Scene([(new, 700), (1, 90)], heads=4, kv_heads=2, hd=64, seed=4, mul=mul).upload()
    have_o, have_l = s.attend()
    want_o, want_l, size = s.expected()
    half = HALF_STEP[BF16]
    assert (np.abs(have_o.astype(np.float64) - want_o) <= half * np.abs(want_o) * (1 + half) + (half + 2.0**-13 * max(1.0, mul)) * size + 2.0**-24).all()
    assert (np.abs(have_l - want_l) <= 2.0**-13 * max(1.0, mul) + 2.0**-23 * np.abs(want_l)).all()


@pytest.mark.parametrize("new", [1, 3, 90])
def test_two_runs_give_the_same_bits(new):
    s = Scene([(new, 2000), (1, 77), (min(new, 30), 555)], heads=8, kv_heads=2, hd=128, seed=6, prefix=0).upload()
    first, second = s.attend(), s.attend()
    assert np.array_equal(first[0].view(np.uint16), second[0].view(np.uint16)) and np.array_equal(first[1], second[1])


def test_scale_of_the_callers_own():
    Scene([(1, 500), (20, 60)], heads=4, kv_heads=2, hd=64, seed=8).upload().check(scale=0.02)


# ---------------------------------------------------------------- what only the device knows

@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("prefix", [0, 40])
def test_a_page_that_is_none(new, prefix):
    """Rows that see a key of such a page get NaN, other rows and sequences are as they would be, and the word says so."""
    seqs = [(new, 400), (new, 300), (1, 64)]
    s = Scene(seqs, heads=4, kv_heads=2, hd=64, page_size=16, seed=3, prefix=prefix)
    for bad in (-1, s.pages, 2**31 - 1, -(2**31)):
        table = s.table.copy()
        table[1, 300 // 16 - 1] = bad  # slots 272 to 287
        s.upload(table=table)
        have_o, have_l = s.attend()
        assert s.error_bits() == 1
        want_o, want_l, size = s.expected()
        sees = np.zeros(s.tokens, bool)
        sees[s.start[1] : s.start[2]] = (300 - new + np.arange(new)) >= 272
        assert np.isnan(have_o[sees].astype(np.float32)).all() and np.isnan(have_l[sees]).all()
        half = HALF_STEP[BF16]
        off = np.abs(have_o[~sees].astype(np.float64) - want_o[~sees])
        assert (off <= half * np.abs(want_o[~sees]) * (1 + half) + (half + 2.0**-13) * size[~sees] + 2.0**-24).all()
        assert (np.abs(have_l[~sees] - want_l[~sees]) <= 2.0**-13 + 2.0**-23 * np.abs(want_l[~sees])).all()


def test_a_prefix_page_that_is_none():
    s = Scene([(1, 40), (2, 30)], heads=4, kv_heads=2, hd=64, page_size=16, seed=3, prefix=100)
    s.prefix_table = s.prefix_table.copy()
    good = s.prefix_table[3]
    s.upload()
    from limn_b200 import runtime

    table = np.append(s.prefix_table, np.int32(NOWHERE))
    table[3] = -5
    s.prefix_dev = runtime.upload(table)
    have_o, have_l = s.attend()
    assert good >= 0 and s.error_bits() == 1 and np.isnan(have_o.astype(np.float32)).all() and np.isnan(have_l).all()


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("what", ["long", "negative", "falling", "wide", "beyond", "before"])
def test_a_sequence_that_cannot_be(what, new):
    """It is left out, its rows as they were; the others are served."""
    seqs = [(new, 200), (new, 100), (new, 300)]
    s = Scene(seqs, heads=4, kv_heads=2, hd=64, page_size=16, seed=3, max_t_q=new)
    start, keys, out_of = list(s.start), [*s.keys, 0], [1]
    if what == "long":
        keys[1] = s.max_pages * 16 + 1
    elif what == "negative":
        keys[1] = -1
    elif what == "falling":
        start[1], out_of = start[2] + 1, [0, 1]  # the first one has too many then, the second fewer than none
    elif what == "wide":
        start[2], out_of = start[2] + 1, [1]  # one token more than max_t_q; the third has one fewer
    elif what == "beyond":
        start[3], out_of = s.tokens + 1, [2]
    else:
        start[0], out_of = -1, [0]
    s.upload(q_start=start, kv_lens=keys)
    have_o, have_l = s.attend()
    assert s.error_bits() == 2
    want_o, want_l, size = s.expected()
    for b in range(3):
        rows = slice(s.start[b], s.start[b + 1])
        if b in out_of:
            rows = slice(s.start[b] + (what == "wide" and b == 2), s.start[b + 1])
            assert (have_o[rows].view(np.uint16) == 0x7FFF).all() and np.isnan(have_l[rows]).all()
        elif not (what == "wide" and b == 2):  # (there the rows moved by one)
            if what == "falling":  # other sequences' rows may be left out as well, but not be wrong
                rows = np.arange(s.tokens)[rows][~np.isnan(have_l[rows, 0])]
            half = HALF_STEP[BF16]
            assert (np.abs(have_o[rows].astype(np.float64) - want_o[rows]) <= half * np.abs(want_o[rows]) * (1 + half) + (half + 2.0**-13) * size[rows] + 2.0**-24).all()
            assert (np.abs(have_l[rows] - want_l[rows]) <= 2.0**-13 + 2.0**-23 * np.abs(want_l[rows])).all()


def test_append_leaves_out_what_has_no_place():
    from limn_b200 import runtime

    s = Scene([(2, 20), (3, 2), (1, 33), (2, 40)], heads=2, kv_heads=1, hd=64, page_size=16, seed=1)
    table, keys = s.table.copy(), [*s.keys, 0]
    table[2, 2] = s.pages  # the third one's token has no page; the second one has more tokens than keys
    keys[3] = 16 * s.max_pages + 1  # the fourth is longer than its table
    s.upload(with_new=False, table=table, kv_lens=keys)
    rng = np.random.default_rng(0)
    k, v = (rng.standard_normal((s.tokens, 1, 64)).astype(np.float32).astype(BF16) for _ in range(2))
    before = s.filled(with_new=False)
    s.step.append(runtime.upload(k), runtime.upload(v))
    runtime.synchronize()
    assert s.error_bits() == 3
    for memory, was, new in ((s.k_dev, before[0], k), (s.v_dev, before[1], v)):
        want = was.copy()
        for t, slot in ((0, 18), (1, 19)):
            want[table[0, slot // 16], slot % 16] = new[t]
        assert np.array_equal(runtime.download(memory, np.uint16, was.shape), want.view(np.uint16))


def test_nothing_to_do():
    s = Scene([(0, 5), (0, 0)], spare_tokens=2).upload()
    s.check()
    empty = Scene([], spare_tokens=2).upload()
    empty.check()
