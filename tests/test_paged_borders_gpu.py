"""A paged key and value cache on the GPU where its documentation leaves room: idle places of a batch, offsets that fall, scores of any size, kernels that give
up in the middle of a call, what one operator leaves for the next. Against the definitions in float64 (paged_scene.py, which derives the tolerances)."""

from __future__ import annotations

import numpy as np
import pytest
from paged_scene import Scene, poison

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


# ---------------------------------------------------------------- giving up in the middle of a call

def test_what_a_kernel_that_gave_up_left_undone_is_not_joined():
    """A wait runs out on another stream while a prompt is being computed: its blocks leave their waits, some of them before they have left the parts that others count
    on. Every row is right or as it was; the workspace holds numbers that would show. The word says who gave up, and the next call is right."""
    from limn_b200 import runtime
    from limn_b200._lib import check, lib

    s = Scene([(20000, 20000)], heads=16, kv_heads=2, hd=128, page_size=64, seed=46).upload()
    good_o, good_l = s.attend()
    q, room = runtime.upload(s.q), s.step.workspace
    main, side, flag = runtime.Stream(), runtime.Stream(), runtime.empty(4, poison=0)
    caught = 0
    for budget in (400_000, 800_000, 1_600_000):  # clock ticks: parts of the prompt's 2 ms
        out, lse = runtime.empty(good_o.nbytes, poison=0x7F), runtime.empty(good_l.nbytes, poison=0x7F)
        check(lib().limn_b200_mem_set(room.ptr, 0x3F, room.nbytes, None), "filling the workspace")
        runtime.synchronize()
        check(lib().limn_b200_wait_probe(budget, flag.ptr, side.handle), "wait probe")
        s.step.attention(q, out, lse, stream=main)
        have_o, have_l = runtime.download(out, np.uint16, good_o.shape), runtime.download(lse, np.uint32, good_l.shape)
        assert runtime.device_status() == 0x57417E57
        as_it_was = (have_o == 0x7F7F).all(-1) & (have_l == 0x7F7F7F7F)
        right = (have_o == good_o.view(np.uint16)).all(-1) & (have_l == good_l.view(np.uint32))
        assert (as_it_was | right).all(), f"{np.count_nonzero(~(as_it_was | right))} rows are neither right nor as they were"
        caught += bool(as_it_was.any() and right.any())
    assert caught, "no attempt met the call in its middle"
    again_o, again_l = s.attend()
    assert np.array_equal(again_o.view(np.uint16), good_o.view(np.uint16)) and np.array_equal(again_l, good_l)
    assert runtime.device_status() == 0


# ---------------------------------------------------------------- one operator after the other

@pytest.mark.parametrize("captured", [False, True], ids=["enqueued", "captured"])
@pytest.mark.parametrize("new, heads", [(1, 8), (3, 8), (60, 8)])
def test_what_append_has_just_written_is_seen_behind_a_prefix_read_once(new, heads, captured):
    """Append, and right behind it the passes over the prefix and over the sequences' own keys, again and again with other tokens in the same arrays and nothing
    between them: every result is, bit by bit, what the call gives when the device is waited for before each."""
    torch = pytest.importorskip("torch")
    from limn_b200 import runtime

    s = Scene([(new, 500), (new, new), (1, 40)] + IDLE, heads=heads, kv_heads=2, hd=128, page_size=16, seed=47, prefix=700).upload(with_new=False)
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(48)
    made = [{name: torch.randn((s.tokens, h, 128), generator=gen, device=dev).to(torch.bfloat16) for name, h in (("q", heads), ("k", 2), ("v", 2))} for _ in range(3)]
    now = {name: torch.zeros_like(x) for name, x in made[0].items()}
    turned, out, lse = torch.zeros_like(now["q"]), torch.zeros_like(now["q"]), torch.zeros((s.tokens, heads), device=dev)
    freqs = 10000.0 ** (-torch.arange(64, dtype=torch.float64, device=dev) / 64)

    def call(stream, between=lambda: None):
        s.step.append(now["k"], now["v"], q=now["q"], q_out=turned, frequencies=freqs, rotated=128, stream=stream)
        between()
        s.step.attention_with_prefix(turned, out, lse, prefix_table=s.prefix_dev, prefix_len=700, stream=stream)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        alone = []
        for x in made:
            for name in now:
                now[name].copy_(x[name])
            side.synchronize()
            call(side.cuda_stream, side.synchronize)
            assert launches() == 3
            side.synchronize()
            alone.append((out.clone(), lse.clone()))
        assert not torch.equal(alone[0][0], alone[1][0])
        side.synchronize()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                call(torch.cuda.current_stream().cuda_stream)
        got = []
        for turn in range(30):
            for name in now:
                now[name].copy_(made[turn % 3][name])
            if captured:
                graph.replay()
            else:
                call(side.cuda_stream)
            got.append((out.clone(), lse.clone()))
        side.synchronize()
    for turn, (o, l) in enumerate(got):
        assert torch.equal(o.view(torch.int16), alone[turn % 3][0].view(torch.int16)) and torch.equal(l, alone[turn % 3][1]), f"turn {turn}"
    assert s.error_bits() == 0
    if captured:
        del graph
    assert runtime.device_status() == 0


# ---------------------------------------------------------------- offsets that fall

@pytest.mark.parametrize("most", [8, 60], ids=["few rows", "many rows"])
@pytest.mark.parametrize("prefix, idle", [(0, 0), (0, 500), (300, 0), (300, 4000)], ids=["alone", "alone, many places", "behind", "behind, read once"])
@pytest.mark.parametrize("start", [[0, 5, 3, 8], [0, 6, 0, 6], [2, 8, 1, 1], [0, 3, 8, 7]], ids=str)
def test_where_offsets_fall_no_row_is_written(start, prefix, idle, most):
    """Sequences that are possible each by itself have tokens in common then: whichever came last would stay. The word says so, run after run, and the next call
    with offsets that rise is right."""
    from limn_b200 import runtime

    s = Scene([(5, 40), (1, 30), (2, 50)] + [(0, 0)] * idle, heads=2, kv_heads=1, hd=64, page_size=16, seed=49, prefix=prefix, max_t_q=most)
    for _ in range(2):
        s.upload(q_start=[*start, *[start[-1]] * idle])
        have_o, have_l = s.attend()
        assert (have_o.view(np.uint16) == 0x7FFF).all() and np.isnan(have_l).all()
        assert s.error_bits() == 2
        assert launches() == (3 if prefix and idle else 2)
        s.upload().check()
    assert runtime.device_status() == 0


# ---------------------------------------------------------------- what is collected while a step is captured

def test_a_batch_may_be_collected_during_a_capture():
    """Its workspace, and pinned memory, are freed in the middle of the capture of another batch's calls, which goes on."""
    torch = pytest.importorskip("torch")
    from limn_b200 import runtime

    s = Scene([(1, 300), (2, 40)], heads=4, kv_heads=2, hd=64, seed=50).upload()
    good_o, good_l = s.attend()
    going = [Scene([(1, 30)], heads=4, kv_heads=2, hd=64, seed=51).upload(), runtime.PinnedArray((100,), np.float32)]
    q, out, lse = runtime.upload(s.q), runtime.empty(good_o.nbytes), runtime.empty(good_l.nbytes)
    runtime.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        going.pop()
        s.step.attention(q, out, lse, stream=torch.cuda.current_stream().cuda_stream)
        going.pop()
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(runtime.download(out, np.uint16, good_o.shape), good_o.view(np.uint16)) and np.array_equal(runtime.download(lse, np.float32, good_l.shape), good_l)
    del graph
    assert runtime.device_status() == 0


# ---------------------------------------------------------------- where the cache is

def test_a_cache_that_is_not_device_memory():
    """Host memory that no kernel could read is refused before anything is launched."""
    import ctypes

    from limn_b200 import runtime
    from limn_b200._lib import last_error, lib

    s = Scene([(1, 30), (2, 40)], heads=4, kv_heads=2, hd=64, seed=52).upload()
    s.check()
    host = np.zeros(s.pages * 16 * 2 * 64 + 8, np.uint16)
    at, pairs = -(-host.ctypes.data // 16) * 16, (ctypes.c_longlong * 8)(256, 64, 256, 64, 128, 64, 128, 64)
    q, out, lse, new = runtime.upload(s.q), runtime.empty(s.q.nbytes), runtime.empty(s.tokens * 4 * 4), runtime.empty(s.tokens * 2 * 64 * 2)
    step, room = s.step._step, s.step.workspace
    on_device, step.k_cache = step.k_cache, at
    for got in (lib().limn_b200_sdpa_paged(s.step._by_ref, q.ptr, out.ptr, lse.ptr, pairs, 1, 0.125, room.ptr, room.nbytes, None),
                lib().limn_b200_sdpa_paged_prefix(s.step._by_ref, q.ptr, out.ptr, lse.ptr, pairs, s.table_dev.ptr, 5, 1, 0.125, room.ptr, room.nbytes, None),
                lib().limn_b200_kv_append(s.step._by_ref, None, new.ptr, new.ptr, None, pairs, None, 0, 0, None)):
        assert got == 1 and "device memory" in last_error() and launches() == 0
    step.k_cache = on_device
    s.check()


# ---------------------------------------------------------------- orders of memory

@pytest.mark.parametrize("hd, hd_v", [(64, 64), (128, 128), (80, 40)])
@pytest.mark.parametrize("new", [1, 3, 70])
@pytest.mark.parametrize("prefix", [0, 40])
def test_heads_outermost_in_queries_results_and_cache(prefix, new, hd, hd_v):
    """(head, token, column) operands and (head, page, slot, column) pages: the largest stride belongs to the head."""
    from limn_b200 import runtime
    from limn_b200.paged import PagedBatch, PagedCache

    s = Scene([(new, 300), (1, 40), (new, new)], heads=8, kv_heads=4, hd=hd, hd_v=hd_v, page_size=16, seed=53, prefix=prefix, spare_tokens=1)
    k, v = (np.ascontiguousarray(x.transpose(2, 0, 1, 3)) for x in s.filled())
    s.upload()
    sides = runtime.upload(k), runtime.upload(v)
    cache = PagedCache(*sides, dtype="bfloat16", pages=s.pages, page_size=16, kv_heads=4, hd=hd, hd_v=hd_v, k_strides=(16 * hd, s.pages * 16 * hd, hd),
                       v_strides=(16 * hd_v, s.pages * 16 * hd_v, hd_v))
    step = PagedBatch(cache, heads=8, batch=3, tokens=s.tokens, max_t_q=new, page_table=s.table_dev, max_pages=s.max_pages, q_start=s.q_start_dev, kv_lens=s.kv_lens_dev, errors=s.errors)
    q = runtime.upload(np.ascontiguousarray(s.q.transpose(1, 0, 2)))
    out, lse = runtime.upload(poison(s.dtype, (8, s.tokens, hd_v))), runtime.upload(np.full((s.tokens, 8), np.nan, np.float32))
    more = {"q_strides": (hd, s.tokens * hd), "out_strides": (hd_v, s.tokens * hd_v)}
    if prefix:
        step.attention_with_prefix(q, out, lse, prefix_table=s.prefix_dev, prefix_len=prefix, **more)
    else:
        step.attention(q, out, lse, **more)
    have = runtime.download(out, np.uint16, (8, s.tokens, hd_v)).view(s.dtype).transpose(1, 0, 2)
    s.compare(np.ascontiguousarray(have), runtime.download(lse, np.float32, (s.tokens, 8)), *s.expected())
    assert s.error_bits() == 0
