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
    ("generation gqa4 128, 4 key heads", BF16, 16, 4, 128, 128, 16, "token", GENERATION),
    ("generation gqa3 64, 5 key heads", F16, 15, 5, 64, 64, 16, "head", GENERATION),
    ("drafts mha 12, 80", F16, 12, 12, 80, 80, 48, "head", DRAFTS),
    ("drafts gqa4 128, 8 key heads", BF16, 32, 8, 128, 128, 16, "token", DRAFTS),
    ("generation, room between heads", BF16, 4, 2, 128, 128, 16, "roomy", GENERATION),
    ("generation, K and V by page", F16, 4, 2, 64, 64, 16, "paired", GENERATION),
    ("prompts, room between heads", BF16, 8, 2, 128, 128, 16, "roomy", PROMPTS),
    ("prompts, K and V by page", BF16, 8, 2, 128, 128, 32, "paired", PROMPTS),
    ("prompts, one key head, room", F16, 4, 1, 128, 128, 8, "roomy", PROMPTS),
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
    k_dev, v_dev = runtime.upload(k), runtime.upload(v)
    s.step.append(k_dev, v_dev)
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


# ---------------------------------------------------------------- many sequences, long ones, far ones

@pytest.mark.parametrize("heads", [2, 32])
@pytest.mark.parametrize("prefix", [0, 20])
def test_more_sequences_than_threads(heads, prefix):
    """700 sequences, some without tokens or keys: every thread of a block adds up several."""
    rng = np.random.default_rng(12)
    seqs = [(int(n), int(n + c)) for n, c in zip(rng.integers(0, 3, 700), rng.integers(0, 40, 700))]
    Scene(seqs, heads=heads, kv_heads=1, hd=64, page_size=8, seed=13, prefix=prefix).upload().check()


@pytest.mark.parametrize("new", [1, 200])
def test_a_long_sequence_among_short_ones(new):
    """One problem is shared by nearly all workers, others share one."""
    Scene([(1, 3), (new, 40000), (1, 17), (2, 2)], heads=2, kv_heads=1, hd=128, page_size=64, seed=14).upload().check()


NARROW = [s for s in SHAPES if max(s[4], s[5]) <= 64 and s[2] // s[3] <= 8 and s[0].startswith("generation")]


@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("shape", NARROW, ids=[s[0] for s in NARROW])
def test_tables_with_room_for_many_keys(shape, prefix):
    """How many keys there can be decides how many warps a block of narrow rows has: here 2^18 to a sequence, and few that there are."""
    _, dtype, heads, kv_heads, hd, hd_v, page_size, order, seqs = shape
    for order in {order, "head"}:
        Scene(seqs, dtype=dtype, heads=heads, kv_heads=kv_heads, hd=hd, hd_v=hd_v, page_size=page_size, order=order, prefix=prefix, spare_tokens=2, seed=37,
              max_pages=(1 << 18) // page_size).upload().check()


@pytest.mark.parametrize("new, heads, hd", [(1, 4, 128), (4, 4, 128), (1, 4, 64), (2, 4, 24)])
@pytest.mark.parametrize("order", ["head", "token"])
def test_long_shares(order, new, heads, hd):
    """64 sequences of 20 000 keys: 44 units of 16 keys and more to every warp of 148 blocks, in pages that they all name."""
    s = Scene([(new, 20000)], heads=heads, kv_heads=1, hd=hd, page_size=64, order=order, seed=35, max_t_q=new)
    many = 64
    s.seqs, s.new, s.keys, s.k, s.v = s.seqs * many, s.new * many, s.keys * many, s.k * many, s.v * many
    s.table, s.start, s.tokens = np.repeat(s.table, many, axis=0), np.arange(many + 1) * new, many * new
    s.q = np.random.default_rng(36).standard_normal((s.tokens, heads, hd)).astype(np.float32).astype(BF16)
    s.upload().check()


@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("new, heads", [(1, 4), (1, 32), (4, 16), (3, 20), (30, 8)])
def test_what_the_workspace_held_is_of_no_concern(new, heads, prefix):
    """The same call again gives the same bits, whatever the workspace held before it."""
    from limn_b200 import runtime
    from limn_b200.paged import PagedBatch

    s = Scene([(new, 6000), (1, 3), (new, 900), (0, 10), (new, 40)], heads=heads, kv_heads=4, hd=128, page_size=16, seed=28, prefix=prefix).upload()
    first = s.check()
    held, size = s.step._held[0], s.step.workspace_bytes
    rng = np.random.default_rng(3)
    for bytes_ in (np.zeros(size, np.uint8), np.full(size, 0xFF, np.uint8), rng.integers(0, 256, size, dtype=np.uint8)):
        memory = runtime.upload(bytes_)
        s.step = PagedBatch(held, heads=heads, batch=5, tokens=s.tokens, max_t_q=s.max_t_q, page_table=s.table_dev, max_pages=s.max_pages, q_start=s.q_start_dev,
                            kv_lens=s.kv_lens_dev, errors=s.errors, workspace=memory, max_prefix=300)
        for _ in range(3):
            again = s.attend()
            assert np.array_equal(first[0].view(np.uint16), again[0].view(np.uint16)) and np.array_equal(first[1], again[1])


def test_a_prefix_far_longer_than_the_rest():
    Scene([(1, 3), (2, 5)], heads=8, kv_heads=2, hd=64, page_size=16, seed=15, prefix=20000).upload().check()
    Scene([(1, 3), (40, 50)], heads=8, kv_heads=2, hd=128, page_size=16, seed=15, prefix=9000).upload().check()


# Behind a prefix that would cost much to read for every sequence, a call reads it once, for the whole batch. Sequences without tokens cost nothing, but how many
# there are counts for that.
IDLE = [(0, 0)] * 4000


def launches() -> int:
    from limn_b200._lib import lib

    return lib().limn_b200_last_launch_count()


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("shape", SHAPES, ids=[s[0] for s in SHAPES])
def test_a_prefix_read_once(shape, causal):
    _, dtype, heads, kv_heads, hd, hd_v, page_size, order, seqs = shape
    s = Scene(seqs + IDLE, dtype=dtype, heads=heads, kv_heads=kv_heads, hd=hd, hd_v=hd_v, page_size=page_size, order=order, prefix=300, spare_tokens=2,
              seed=11, row_room=8).upload()
    s.check(causal=causal)
    assert launches() == 3


@pytest.mark.parametrize("length", [8, 15, 16, 17, 120, 127, 128, 129, 255, 256, 257, 1024])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("once", [False, True], ids=["for each", "once"])
def test_every_length_of_a_prefix(length, new, once):
    """Where a prefix ends inside a unit or a tile of keys, beside sequences that have no keys, few, or see none of their own."""
    s = Scene([(new, new), (1, 0), (new, new + 100), (2, 1)] + IDLE * (10 if once else 0), heads=8, kv_heads=2, hd=64, page_size=8, seed=length, prefix=length).upload()
    s.check()
    assert launches() == (3 if once else 2)
    s.check(causal=False)


@pytest.mark.parametrize("heads", [1, 2, 4])
def test_more_tokens_than_keys_behind_a_prefix_read_once(heads):
    s = Scene([(5, 3), (1, 0), (40, 2), (2, 200)] + IDLE, heads=heads, kv_heads=1, hd=64, seed=2, prefix=700).upload()
    s.check()
    assert launches() == 3


@pytest.mark.parametrize("idle", [[], IDLE], ids=["for each", "once"])
@pytest.mark.parametrize("new", [1, 60])
def test_pages_that_are_none_behind_a_prefix(new, idle):
    """One of a sequence's own: the rows that see it. One of the prefix: all rows."""
    from limn_b200 import runtime

    s = Scene([(new, 400), (new, 300), (1, 64)] + idle, heads=4, kv_heads=2, hd=64, page_size=16, seed=3, prefix=700)
    table = s.table.copy()
    table[1, 300 // 16 - 1] = -9  # slots 272 to 287
    s.upload(table=table)
    have_o, have_l = s.attend()
    assert s.error_bits() == 1 and launches() == (3 if idle else 2)
    want_o, want_l, size = s.expected()
    sees = np.zeros(s.tokens, bool)
    sees[s.start[1] : s.start[2]] = (300 - new + np.arange(new)) >= 272
    assert np.isnan(have_o[sees].astype(np.float32)).all() and np.isnan(have_l[sees]).all()
    half = HALF_STEP[BF16]
    off = np.abs(have_o[~sees].astype(np.float64) - want_o[~sees])
    assert (off <= half * np.abs(want_o[~sees]) * (1 + half) + (half + 2.0**-13) * size[~sees] + 2.0**-24).all()
    assert (np.abs(have_l[~sees] - want_l[~sees]) <= 2.0**-13 + 2.0**-23 * np.abs(want_l[~sees])).all()
    for which in (0, 20, 43):  # the last one holds 12 keys
        bad = np.append(s.prefix_table, np.int32(NOWHERE))
        bad[which] = s.pages
        s.upload()
        s.prefix_dev = runtime.upload(bad)
        have_o, have_l = s.attend()
        assert s.error_bits() == 1 and np.isnan(have_o.astype(np.float32)).all() and np.isnan(have_l).all()


@pytest.mark.parametrize("new, heads", [(1, 4), (1, 32), (4, 16), (3, 20), (30, 8)])
def test_what_the_workspace_held_is_of_no_concern_to_a_prefix_read_once(new, heads):
    from limn_b200 import runtime
    from limn_b200.paged import PagedBatch

    s = Scene([(new, 600), (1, 3), (new, 900), (0, 10), (new, 40)] + IDLE, heads=heads, kv_heads=4, hd=128, page_size=16, seed=28, prefix=300).upload()
    first = s.check()
    assert launches() == 3
    held, size = s.step._held[0], s.step.workspace_bytes
    rng = np.random.default_rng(3)
    for bytes_ in (np.full(size, 0xFF, np.uint8), rng.integers(0, 256, size, dtype=np.uint8)):
        memory = runtime.upload(bytes_)
        s.step = PagedBatch(held, heads=heads, batch=len(s.seqs), tokens=s.tokens, max_t_q=s.max_t_q, page_table=s.table_dev, max_pages=s.max_pages,
                            q_start=s.q_start_dev, kv_lens=s.kv_lens_dev, errors=s.errors, workspace=memory)
        for _ in range(3):
            again = s.attend()
            assert np.array_equal(first[0].view(np.uint16), again[0].view(np.uint16)) and np.array_equal(first[1], again[1])


def test_a_workspace_serves_a_prefix_of_any_length():
    """It is sized for one key: as much as any longer one needs."""
    from limn_b200.paged import PagedBatch

    s = Scene([(1, 60), (30, 40)] + IDLE, heads=4, kv_heads=2, hd=64, seed=29, prefix=900).upload()
    s.step = PagedBatch(s.step._held[0], heads=4, batch=len(s.seqs), tokens=s.tokens, max_t_q=30, page_table=s.table_dev, max_pages=s.max_pages,
                        q_start=s.q_start_dev, kv_lens=s.kv_lens_dev, errors=s.errors, first_position=900)
    s.check()
    assert launches() == 3


def test_standing_down_behind_a_prefix_read_once():
    from limn_b200 import runtime
    from limn_b200._lib import check, lib

    s = Scene([(60, 500), (1, 70)] + IDLE, heads=4, kv_heads=2, hd=64, seed=27, prefix=300).upload()
    s.check()
    assert launches() == 3
    flag = runtime.empty(4, poison=0)
    check(lib().limn_b200_wait_probe(20000, flag.ptr, None), "wait probe")
    have_o, have_l = s.attend()
    assert (have_o.view(np.uint16) == 0x7FFF).all() and np.isnan(have_l).all()
    assert runtime.device_status() == 0x57417E57
    s.check()


@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_31_bits(new):
    """Pages 2^27 elements apart: the last one begins 2^31 elements, 2^32 bytes, in."""
    from limn_b200 import runtime
    from limn_b200._lib import check, lib
    from limn_b200.paged import PagedBatch, PagedCache

    s = Scene([(new, 100), (1, 30)], heads=4, kv_heads=1, hd=64, page_size=16, seed=16, spare_pages=10)
    apart = 1 << 27
    assert s.pages == 19 and int(s.table[s.table < s.pages].max()) * apart >= 2**31
    k, v = s.filled(with_new=False)
    far = [runtime.DeviceBuffer(2 * (apart * (s.pages - 1) + 16 * 64)) for _ in range(2)]
    for host, memory in ((k, far[0]), (v, far[1])):
        for page in range(s.pages):
            check(lib().limn_b200_copy_h2d(memory.ptr + 2 * apart * page, np.ascontiguousarray(host[page]).ctypes.data, 16 * 64 * 2, None), "uploading a page")
            runtime.synchronize()
    s.upload()
    cache = PagedCache(*far, dtype="bfloat16", pages=s.pages, page_size=16, kv_heads=1, hd=64, k_strides=(apart, 64, 64), v_strides=(apart, 64, 64))
    s.step = PagedBatch(cache, heads=4, batch=2, tokens=s.tokens, max_t_q=s.max_t_q, page_table=s.table_dev, max_pages=s.max_pages, q_start=s.q_start_dev,
                        kv_lens=s.kv_lens_dev, errors=s.errors)
    new_k = np.concatenate([s.k[b][-n:] for b, n in enumerate(s.new)])
    new_v = np.concatenate([s.v[b][-n:] for b, n in enumerate(s.new)])
    new_k, new_v = runtime.upload(new_k), runtime.upload(new_v)
    s.step.append(new_k, new_v)  # not turned: what the scene has
    s.check()


# ---------------------------------------------------------------- as they are used: together, captured, on streams

def _frequencies(rotated):
    return 10000.0 ** (-np.arange(rotated // 2) / (rotated // 2))


@pytest.mark.parametrize("hd", [64, 128])
def test_a_prompt_and_then_token_by_token(hd):
    """A model's layer over the life of two sequences: the prompt enters the cache in one step, then every step brings a token to
    each (and none to the first in the third). In the end every row is what one causal pass of the library over all tokens gives, up
    to the rounding of the weights on either side, which the definitions in float64 measure."""
    from limn_b200 import runtime
    from limn_b200._lib import check, lib
    from limn_b200.paged import PagedBatch, PagedCache

    rng = np.random.default_rng(17)
    heads, kv_heads, page_size, max_pages, pages = 8, 2, 16, 12, 30
    steps = [[100, 37], [1, 1], [1, 1], [0, 1], [1, 1], [1, 1], [3, 2]]
    total = [sum(x) for x in zip(*steps)]
    made = [{name: rng.standard_normal((t, h, hd)).astype(np.float32).astype(BF16) for name, h in (("q", heads), ("k", kv_heads), ("v", kv_heads))} for t in total]
    table = rng.permutation(pages)[: 2 * max_pages].reshape(2, max_pages).astype(np.int32)
    k_dev, v_dev = (runtime.upload(poison(BF16, (pages, page_size, kv_heads, hd))) for _ in range(2))
    cache = PagedCache(k_dev, v_dev, dtype="bfloat16", pages=pages, page_size=page_size, kv_heads=kv_heads, hd=hd)
    table_dev, errors, freqs = runtime.upload(table), runtime.upload(np.zeros(1, np.uint32)), runtime.upload(_frequencies(hd))
    done, got, turned_q = [0, 0], [[], []], [[], []]
    for new in steps:
        start = np.array([0, new[0], sum(new)], np.int32)
        step = PagedBatch(cache, heads=heads, batch=2, tokens=sum(new), max_t_q=max(new), page_table=table_dev, max_pages=max_pages, q_start=runtime.upload(start),
                          kv_lens=runtime.upload(np.array([d + n for d, n in zip(done, new)], np.int32)), errors=errors)
        now = {name: runtime.upload(np.concatenate([made[b][name][done[b] : done[b] + new[b]] for b in range(2)])) for name in "qkv"}
        out, lse = runtime.empty(sum(new) * heads * hd * 2), runtime.empty(sum(new) * heads * 4)
        step.append(now["k"], now["v"], q=now["q"], q_out=now["q"], frequencies=freqs, rotated=hd)
        step.attention(now["q"], out, lse)
        rows, turned = (runtime.download(x, np.uint16, (sum(new), heads, hd)).view(BF16) for x in (out, now["q"]))
        for b in range(2):
            got[b].append(rows[start[b] : start[b + 1]])
            turned_q[b].append(turned[start[b] : start[b + 1]])
            done[b] += new[b]
    assert runtime.download(errors, np.uint32, (1,))[0] == 0
    k_all, v_all = (runtime.download(x, np.uint16, (pages, page_size, kv_heads, hd)).view(BF16) for x in (k_dev, v_dev))
    for b, t in enumerate(total):
        slots = np.arange(t)
        k, v = (x[table[b][slots // page_size], slots % page_size] for x in (k_all, v_all))
        q, rows = np.concatenate(turned_q[b]), np.concatenate(got[b])
        wide = np.repeat(k, heads // kv_heads, axis=1), np.repeat(v, heads // kv_heads, axis=1)
        by_head = [runtime.upload(np.ascontiguousarray(x.transpose(1, 0, 2))) for x in (q, *wide)]
        out, lse = runtime.empty(rows.nbytes), runtime.empty(heads * t * 4)
        check(lib().limn_b200_sdpa_fwd(*(x.ptr for x in by_head), None, out.ptr, lse.ptr, 2, heads, t, t, hd, hd, 1, hd**-0.5, None), "sdpa")
        dense = runtime.download(out, np.uint16, (heads, t, hd)).view(BF16).transpose(1, 0, 2).astype(np.float64)
        s = np.einsum("thd,jhd->thj", q.astype(np.float64), wide[0].astype(np.float64)) * hd**-0.5
        s[np.broadcast_to(np.arange(t)[:, None, None] < np.arange(t), s.shape)] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        size = np.einsum("thj,jhd->thd", p, np.abs(wide[1].astype(np.float64)))
        half = HALF_STEP[BF16]
        # either side is off by half a step of its value and of the weights, and by 2^-13 of them (paged_scene.py)
        assert (np.abs(rows.astype(np.float64) - dense) <= 2 * (half * np.abs(dense) * (1 + 2 * half) + (half + 2.0**-13) * size * (1 + half)) + 2.0**-23).all()


@pytest.mark.parametrize("new", [1, 30])
def test_a_captured_step_follows_its_arrays(new):
    """append and both attentions in one graph, replayed after offsets, lengths, tables, pages and operands have changed in place."""
    torch = pytest.importorskip("torch")
    from limn_b200 import runtime
    from limn_b200.paged import PagedBatch, PagedCache

    scenes = [Scene([(new, 300), (0, 40), (new, 90)], heads=4, kv_heads=2, hd=64, seed=20, prefix=50, max_pages=20, max_t_q=new),
              Scene([(new, new), (new, 200), (0, 0)], heads=4, kv_heads=2, hd=64, seed=21, prefix=50, max_pages=20, max_t_q=new)]
    pages = max(s.pages for s in scenes)
    dev = torch.device("cuda")
    k_dev, v_dev = (torch.zeros((pages, 16, 2, 64), dtype=torch.bfloat16, device=dev) for _ in range(2))
    q, out = (torch.zeros((2 * new, 4, 64), dtype=torch.bfloat16, device=dev) for _ in range(2))
    k_new, v_new = (torch.zeros((2 * new, 2, 64), dtype=torch.bfloat16, device=dev) for _ in range(2))
    out_prefix, lse, lse_prefix = torch.zeros_like(out), torch.zeros((2 * new, 4), device=dev), torch.zeros((2 * new, 4), device=dev)
    ints = {name: torch.zeros(shape, dtype=torch.int32, device=dev) for name, shape in (("table", (3, 20)), ("q_start", (4,)), ("kv_lens", (3,)), ("prefix", (4,)), ("errors", (1,)))}
    cache = PagedCache(k_dev, v_dev, dtype="bfloat16", pages=pages, page_size=16, kv_heads=2, hd=64)
    step = PagedBatch(cache, heads=4, batch=3, tokens=2 * new, max_t_q=new, page_table=ints["table"], max_pages=20, q_start=ints["q_start"], kv_lens=ints["kv_lens"],
                      errors=ints["errors"], first_position=50, max_prefix=50)

    def bits(x):
        return torch.from_numpy(x.view(np.int16).copy()).to(dev).view(torch.bfloat16)

    def load(s):
        k, v = s.filled(with_new=False)
        k_dev[: s.pages].copy_(bits(k)), v_dev[: s.pages].copy_(bits(v))
        q.copy_(bits(s.q))
        for memory, rows in ((k_new, s.k), (v_new, s.v)):
            memory.copy_(bits(np.concatenate([rows[b][len(rows[b]) - n :] for b, n in enumerate(s.new)])))
        for name, x in (("table", s.table), ("q_start", s.start), ("kv_lens", s.keys), ("prefix", s.prefix_table)):
            ints[name].copy_(torch.as_tensor(np.asarray(x, np.int32)))

    def call(stream):
        step.append(k_new, v_new, stream=stream)
        step.attention(q, out, lse, stream=stream)
        step.attention_with_prefix(q, out_prefix, lse_prefix, prefix_table=ints["prefix"], prefix_len=50, stream=stream)

    load(scenes[0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(side.cuda_stream)  # once before the capture
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(torch.cuda.current_stream().cuda_stream)
    for s in (scenes[1], scenes[0], scenes[1]):
        load(s)
        for x in (out, out_prefix):
            x.view(torch.int16).fill_(0x7FFF)
        lse.fill_(float("nan")), lse_prefix.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for prefix, o, l in ((50, out_prefix, lse_prefix), (0, out, lse)):
            whole = s.prefix, s.prefix_k, s.prefix_v
            if prefix == 0:
                s.prefix, s.prefix_k, s.prefix_v = 0, s.prefix_k[:0], s.prefix_v[:0]
            s.compare(o.view(torch.int16).cpu().numpy().view(BF16), l.cpu().numpy(), *s.expected())
            s.prefix, s.prefix_k, s.prefix_v = whole
    assert ints["errors"].item() == 0
    del graph
    assert runtime.device_status() == 0


def test_two_batches_on_two_streams():
    """Steps with workspaces of their own overlap without touching one another."""
    from limn_b200 import runtime

    scenes = [Scene([(1, 5000), (1, 70), (1, 900)], heads=8, kv_heads=2, hd=128, seed=22).upload(),
              Scene([(60, 3000), (1, 70)], heads=8, kv_heads=2, hd=64, seed=23, prefix=400).upload()]
    alone = [s.attend() for s in scenes]
    streams = [runtime.Stream(), runtime.Stream()]
    held = []
    for _ in range(20):
        for s, stream in zip(scenes, streams):
            q = runtime.upload(s.q) if not hasattr(s, "q_dev") else s.q_dev
            s.q_dev = q
            out, lse = runtime.empty(s.tokens * s.heads * s.hd * 2, poison=None), runtime.empty(s.tokens * s.heads * 4, poison=None)
            if s.prefix:
                s.step.attention_with_prefix(q, out, lse, prefix_table=s.prefix_dev, prefix_len=s.prefix, stream=stream)
            else:
                s.step.attention(q, out, lse, stream=stream)
            held.append((s, out, lse))
    runtime.synchronize()
    for s, out, lse in held:
        want_o, want_l = alone[scenes.index(s)]
        assert np.array_equal(runtime.download(out, np.uint16, want_o.shape), want_o.view(np.uint16))
        assert np.array_equal(runtime.download(lse, np.float32, want_l.shape), want_l)


def test_sequences_may_share_pages():
    s = Scene([(1, 60), (1, 60), (1, 33)], heads=4, kv_heads=2, hd=64, seed=24)
    s.table[1], s.k[1], s.v[1] = s.table[0], s.k[0], s.v[0]
    s.upload().check()


def test_no_word_for_errors():
    from limn_b200.paged import PagedBatch

    s = Scene([(1, 60), (30, 40)], heads=4, kv_heads=2, hd=64, seed=25)
    table = s.table.copy()
    table[0, 1] = -7
    s.upload(table=table)
    held = s.step._held
    s.step = PagedBatch(held[0], heads=4, batch=2, tokens=s.tokens, max_t_q=30, page_table=s.table_dev, max_pages=s.max_pages, q_start=s.q_start_dev, kv_lens=s.kv_lens_dev)
    have_o, _ = s.attend()
    assert np.isnan(have_o[0].astype(np.float32)).all() and np.isfinite(have_o[1:].astype(np.float32)).all() and s.error_bits() == 0


@pytest.mark.parametrize("new", [1, 40])
def test_strides_that_are_never_stepped(new):
    """One page, one head: their strides may be anything, 0 too."""
    from limn_b200 import runtime
    from limn_b200.paged import PagedBatch, PagedCache

    s = Scene([(new, 50)], heads=1, kv_heads=1, hd=128, page_size=64, seed=30, spare_pages=0).upload()
    s.check()
    cache = PagedCache(s.k_dev, s.v_dev, dtype="bfloat16", pages=1, page_size=64, kv_heads=1, hd=128, k_strides=(0, 0, 128), v_strides=(0, 0, 128))
    step = PagedBatch(cache, heads=1, batch=1, tokens=new, max_t_q=new, page_table=s.table_dev, max_pages=1, q_start=s.q_start_dev, kv_lens=s.kv_lens_dev, max_prefix=0)
    q = runtime.upload(s.q)
    out, lse = runtime.upload(poison(BF16, (new, 1, 128))), runtime.upload(np.full((new, 1), np.nan, np.float32))
    step.attention(q, out, lse, q_strides=(128, 0), out_strides=(128, 0))
    runtime.synchronize()
    s.compare(runtime.download(out, np.uint16, (new, 1, 128)).view(BF16), runtime.download(lse, np.float32, (new, 1)), *s.expected())


@pytest.mark.parametrize("new", [1, 40])
def test_key_heads_that_are_the_same(new):
    """A head stride of 0: all key heads read one."""
    from limn_b200.paged import PagedBatch, PagedCache

    s = Scene([(new, 300), (1, 40)], heads=4, kv_heads=1, hd=64, page_size=16, seed=31).upload()
    want, _ = s.check()
    cache = PagedCache(s.k_dev, s.v_dev, dtype="bfloat16", pages=s.pages, page_size=16, kv_heads=2, hd=64, k_strides=(1024, 0, 64), v_strides=(1024, 0, 64))
    s.step = PagedBatch(cache, heads=4, batch=2, tokens=s.tokens, max_t_q=new, page_table=s.table_dev, max_pages=s.max_pages, q_start=s.q_start_dev, kv_lens=s.kv_lens_dev)
    s.check()


@pytest.mark.parametrize("captured", [False, True], ids=["enqueued", "captured"])
def test_calls_of_all_kinds_one_after_the_other_on_one_workspace(captured):
    """Few rows and many, without a prefix, behind one that is read for each sequence and behind one that is read once, with nothing between them: each begins under the one in front
    of it, and they have one workspace. Every result is, bit by bit, what the call gives alone."""
    torch = pytest.importorskip("torch")
    from limn_b200 import runtime
    from limn_b200.paged import PagedBatch

    new = {"few": [(1, 900), (2, 40), (1, 3000)], "many": [(90, 700), (1, 2000), (40, 60)]}
    scenes = [Scene(new[kind] + idle, heads=8, kv_heads=2, hd=128, seed=40 + i, prefix=prefix).upload()
              for i, (kind, prefix, idle) in enumerate([("few", 0, []), ("many", 0, []), ("few", 300, []), ("many", 300, IDLE), ("few", 300, IDLE), ("many", 300, [])])]
    alone, calls = [], []
    largest = max(scenes, key=lambda s: s.step.workspace_bytes).step.workspace
    for s, kernels in zip(scenes, (2, 2, 2, 3, 3, 2), strict=True):
        alone.append(s.check())
        assert launches() == kernels
        s.step = PagedBatch(s.step._held[0], heads=8, batch=len(s.seqs), tokens=s.tokens, max_t_q=s.max_t_q, page_table=s.table_dev, max_pages=s.max_pages,
                            q_start=s.q_start_dev, kv_lens=s.kv_lens_dev, errors=s.errors, workspace=largest)
        calls.append((runtime.upload(s.q), runtime.upload(poison(BF16, (2, s.tokens, 8, 128))), runtime.upload(np.full((2, s.tokens, 8), np.nan, np.float32))))

    def all_of_them(stream):
        for turn in range(2):
            for s, (q, out, lse) in zip(scenes, calls, strict=True):
                o, l = out.ptr + turn * s.tokens * 8 * 128 * 2, lse.ptr + turn * s.tokens * 8 * 4
                if s.prefix:
                    s.step.attention_with_prefix(q, o, l, prefix_table=s.prefix_dev, prefix_len=s.prefix, stream=stream)
                else:
                    s.step.attention(q, o, l, stream=stream)

    runtime.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        if captured:
            with torch.cuda.graph(graph, stream=side):
                all_of_them(torch.cuda.current_stream().cuda_stream)
            graph.replay()
            graph.replay()
        else:
            all_of_them(side.cuda_stream)
    side.synchronize()
    for s, (_, out, lse), (want_o, want_l) in zip(scenes, calls, alone, strict=True):
        have_o, have_l = runtime.download(out, np.uint16, (2, s.tokens, 8, 128)), runtime.download(lse, np.float32, (2, s.tokens, 8))
        for turn in range(2):
            assert np.array_equal(have_o[turn], want_o.view(np.uint16)) and np.array_equal(have_l[turn], want_l)
    del graph
    assert runtime.device_status() == 0


def test_layers_share_a_workspace():
    """Calls that follow one another on a stream: batches over the caches of two layers, one workspace; and one that is too small."""
    from limn_b200.paged import PagedBatch

    first = Scene([(1, 900), (40, 300)], heads=8, kv_heads=2, hd=64, seed=32).upload()
    second = Scene([(1, 900), (40, 300)], heads=8, kv_heads=2, hd=64, seed=33).upload()
    more = dict(heads=8, batch=2, tokens=41, max_t_q=40, max_pages=second.max_pages, page_table=second.table_dev, q_start=second.q_start_dev, kv_lens=second.kv_lens_dev)
    second.step = PagedBatch(second.step._held[0], workspace=first.step.workspace, **more)
    for _ in range(2):
        first.check()
        second.check()
    with pytest.raises(ValueError, match="workspace"):
        PagedBatch(second.step._held[0], workspace=first.errors, **more)


def test_launches_and_workspace():
    import ctypes

    from limn_b200._lib import last_error, lib

    s = Scene([(1, 60), (2, 40)], heads=4, kv_heads=2, hd=64, seed=26, prefix=20).upload()
    for s.prefix in (20, 0):
        s.attend()
        assert lib().limn_b200_last_launch_count() == 2
    need = ctypes.c_ulonglong()
    assert lib().limn_b200_sdpa_paged_workspace(s.step._by_ref, 0, ctypes.byref(need)) == 0 and need.value > 0
    with_prefix = ctypes.c_ulonglong()
    assert lib().limn_b200_sdpa_paged_workspace(s.step._by_ref, 20, ctypes.byref(with_prefix)) == 0 and with_prefix.value > need.value
    strides = (ctypes.c_longlong * 4)(256, 64, 256, 64)
    q = 256
    for workspace, size in ((None, need.value), (256, need.value - 1), (0, 0)):
        assert lib().limn_b200_sdpa_paged(s.step._by_ref, q, q, q, strides, 1, 0.125, workspace, size, None) == 1 and "workspace" in last_error()
    assert lib().limn_b200_last_launch_count() == 0


def test_paged_kernels_stand_down_after_a_wait_that_ran_out():
    """While the status word is set, the kernels that wait, and what joins their results, write nothing; the next call after it has been read is right."""
    from limn_b200 import runtime
    from limn_b200._lib import check, lib

    s = Scene([(60, 500), (1, 70)], heads=4, kv_heads=2, hd=64, seed=27, prefix=0).upload()
    behind = Scene([(60, 500), (1, 70)], heads=4, kv_heads=2, hd=64, seed=27, prefix=90).upload()
    for scene in (s, behind):
        scene.check()
        flag = runtime.empty(4, poison=0)
        check(lib().limn_b200_wait_probe(20000, flag.ptr, None), "wait probe")
        have_o, have_l = scene.attend()
        assert (have_o.view(np.uint16) == 0x7FFF).all() and np.isnan(have_l).all()
        assert runtime.device_status() == 0x57417E57
        scene.check()
    assert runtime.device_status() == 0
