"""What a paged cache refuses, and how its binding packs a call: no GPU."""

from __future__ import annotations

import ctypes

import pytest

ONE = 256  # any aligned, non-null address; the checks below fail before anything is dereferenced


def step(**other):
    from limn_b200._lib import Paged

    values = dict(k_cache=ONE, v_cache=ONE, page_table=ONE, q_start=ONE, kv_lens=ONE, errors=None,
                  k_strides=(ctypes.c_longlong * 3)(2048, 64, 128), v_strides=(ctypes.c_longlong * 3)(2048, 64, 128), dtype=2, batch=3, heads=4,
                  kv_heads=2, hd=64, hd_v=64, page_size=16, pages=10, max_pages=4, tokens=5, max_t_q=2, first_position=0)
    values.update(other)
    return Paged(**values)


def triple(*x):
    return (ctypes.c_longlong * 3)(*x)


REFUSED = [
    # code, words of the message, changed fields
    (1, "dtype", {"dtype": 9}),
    (2, "f16/bf16", {"dtype": 0}),
    (2, "f16/bf16", {"dtype": 3}),
    (1, "positive", {"batch": -1}),
    (1, "positive", {"tokens": -1}),
    (1, "positive", {"max_t_q": 0}),
    (1, "positive", {"heads": 0}),
    (1, "positive", {"kv_heads": 0}),
    (1, "positive", {"hd": 0}),
    (1, "positive", {"hd_v": -8}),
    (1, "positive", {"page_size": 0}),
    (1, "positive", {"pages": 0}),
    (1, "positive", {"max_pages": 0}),
    (1, "no multiple", {"heads": 5}),
    (1, "first position", {"first_position": -1}),
    (2, "multiples of 8", {"hd": 60}),
    (2, "up to 128", {"hd": 136}),
    (2, "up to 128", {"hd_v": 256}),
    (2, "page size", {"page_size": 4}),
    (2, "page size", {"page_size": 1}),
    (2, "at most 128", {"heads": 258, "kv_heads": 2}),
    (2, "31 bits", {"max_pages": 1 << 27, "page_size": 16}),
    (2, "31 bits", {"max_pages": 4, "first_position": 0x7FFFFFF0}),
    (2, "31 bits", {"tokens": 1 << 28, "heads": 16}),
    (2, "31 bits", {"batch": 0x7FFFFFFF}),
    (2, "counts", {"batch": 1 << 20, "tokens": 1 << 20, "heads": 128, "kv_heads": 128, "max_pages": 1 << 20}),
    (1, "strides", {"k_strides": triple(2048, 60, 128)}),
    (1, "strides", {"v_strides": triple(-2048, 64, 128)}),
]
POINTERS = [
    (1, "null", {"k_cache": None}),
    (1, "null", {"v_cache": None}),
    (1, "null", {"page_table": None}),
    (1, "null", {"q_start": None}),
    (1, "null", {"kv_lens": None}),
    (1, "aligned", {"k_cache": ONE + 8}),
    (1, "aligned", {"v_cache": ONE + 2}),
    (1, "aligned", {"page_table": ONE + 2}),
    (1, "aligned", {"q_start": ONE + 1}),
    (1, "aligned", {"kv_lens": ONE + 2}),
    (1, "aligned", {"errors": ONE + 3}),
]


@pytest.mark.parametrize("code, words, other", REFUSED + POINTERS)
@pytest.mark.parametrize("op", ["append", "attention", "prefix"])
def test_a_step_that_cannot_be_is_refused(op, code, words, other):
    from limn_b200._lib import last_error, lib

    L, s = lib(), step(**other)
    pairs = (ctypes.c_longlong * 8)(256, 64, 256, 64, 128, 64, 128, 64)
    if op == "append":
        got = L.limn_b200_kv_append(ctypes.byref(s), ONE, ONE, ONE, ONE, pairs, ONE, 64, 0, None)
    elif op == "attention":
        got = L.limn_b200_sdpa_paged(ctypes.byref(s), ONE, ONE, ONE, pairs, 1, 0.125, ONE, 1 << 40, None)
    else:
        got = L.limn_b200_sdpa_paged_prefix(ctypes.byref(s), ONE, ONE, ONE, pairs, ONE, 30, 1, 0.125, ONE, 1 << 40, None)
    assert got == code and words in last_error(), last_error()
    assert L.limn_b200_last_launch_count() == 0


@pytest.mark.parametrize("code, words, other", REFUSED)
def test_the_workspace_of_a_step_that_cannot_be(code, words, other):
    from limn_b200._lib import last_error, lib

    need = ctypes.c_ulonglong()
    assert lib().limn_b200_sdpa_paged_workspace(ctypes.byref(step(**other)), 0, ctypes.byref(need)) == code and words in last_error()


def test_calls_that_cannot_be():
    from limn_b200._lib import last_error, lib

    L, s = lib(), ctypes.byref(step())
    pairs = (ctypes.c_longlong * 8)(256, 64, 256, 64, 128, 64, 128, 64)
    append = lambda *, q=ONE, k=ONE, v=ONE, q_out=ONE, strides=pairs, freqs=ONE, rotated=64, pairing=0: L.limn_b200_kv_append(s, q, k, v, q_out, strides, freqs, rotated, pairing, None)  # noqa: E731
    for code, words, other in ((1, "null", {"k": None}), (1, "null", {"v": None}), (1, "null", {"q": None}), (1, "null", {"q_out": None}), (1, "null", {"strides": None}),
                               (1, "rotated", {"rotated": 72}), (1, "rotated", {"rotated": -8}), (1, "rotated", {"rotated": 12}), (1, "frequencies", {"freqs": None}),
                               (1, "pairing", {"pairing": 2}), (1, "aligned", {"q": ONE + 4}), (1, "aligned", {"k": ONE + 8}), (1, "aligned", {"freqs": ONE + 4}),
                               (1, "strides", {"strides": (ctypes.c_longlong * 8)(256, 64, 256, 64, 128, 60, 128, 64)}),
                               (1, "strides", {"strides": (ctypes.c_longlong * 8)(-256, 64, 256, 64, 128, 64, 128, 64)})):
        assert append(**other) == code and words in last_error(), (other, last_error())
    # without queries their strides are not read
    assert L.limn_b200_kv_append(ctypes.byref(step(tokens=0)), None, ONE, ONE, None, (ctypes.c_longlong * 8)(1, 1, 1, 1, 128, 64, 128, 64), ONE, 64, 0, None) == 0

    attend = lambda *, q=ONE, out=ONE, lse=ONE, strides=pairs, scale=0.125: L.limn_b200_sdpa_paged(s, q, out, lse, strides, 1, scale, ONE, 1 << 40, None)  # noqa: E731
    for code, words, other in ((1, "null", {"q": None}), (1, "null", {"out": None}), (1, "null", {"lse": None}), (1, "null", {"strides": None}), (1, "aligned", {"q": ONE + 8}),
                               (1, "aligned", {"out": ONE + 2}), (1, "aligned", {"lse": ONE + 2}), (2, "scale", {"scale": 0.0}), (2, "scale", {"scale": -0.1}), (2, "scale", {"scale": float("nan")}),
                               (2, "scale", {"scale": float("inf")}), (2, "scale", {"scale": 1e-46}), (1, "strides", {"strides": (ctypes.c_longlong * 4)(256, 64, 256, 4)})):
        assert attend(**other) == code and words in last_error(), (other, last_error())
    prefix = lambda table, length: L.limn_b200_sdpa_paged_prefix(s, ONE, ONE, ONE, pairs, table, length, 1, 0.125, ONE, 1 << 40, None)  # noqa: E731
    assert prefix(ONE + 2, 10) == 1 and "aligned" in last_error()
    many = ctypes.byref(step(batch=1 << 20, tokens=1 << 20))
    assert L.limn_b200_sdpa_paged_prefix(many, ONE, ONE, ONE, pairs, ONE, 0x7FFF0000, 1, 0.125, ONE, 1 << 40, None) == 2 and "counts" in last_error()
    assert prefix(None, 10) == 1 and prefix(ONE, 0) == 1 and prefix(ONE, -4) == 1 and "prefix" in last_error()
    assert L.limn_b200_sdpa_paged(None, ONE, ONE, ONE, pairs, 1, 0.125, ONE, 1 << 40, None) == 1 and "null step" in last_error()
    assert L.limn_b200_sdpa_paged_workspace(s, 0, None) == 1 and L.limn_b200_sdpa_paged_workspace(s, -1, ctypes.byref(ctypes.c_ulonglong())) == 1


def test_a_step_of_nothing_launches_nothing():
    from limn_b200._lib import last_error, lib

    L = lib()
    pairs = (ctypes.c_longlong * 8)(256, 64, 256, 64, 128, 64, 128, 64)
    for nothing in ({"tokens": 0}, {"batch": 0}):
        s = ctypes.byref(step(**nothing))
        assert L.limn_b200_kv_append(s, ONE, ONE, ONE, ONE, pairs, ONE, 64, 0, None) == 0
        assert L.limn_b200_sdpa_paged(s, ONE, ONE, ONE, pairs, 1, 0.125, None, 0, None) == 0
        assert L.limn_b200_sdpa_paged_prefix(s, ONE, ONE, ONE, pairs, ONE, 5, 1, 0.125, None, 0, None) == 0
        assert L.limn_b200_last_launch_count() == 0 and last_error() == ""


def test_the_binding_reads_addresses_and_strides():
    from limn_b200 import paged

    class Buffer:
        ptr = 4096

    class Tensor:
        def data_ptr(self):
            return 8192

    assert [paged._address(x) for x in (None, 512, Buffer(), Tensor(), Buffer())] == [None, 512, 4096, 8192, 4096]
    with pytest.raises(AttributeError):
        paged._address("nothing of the kind")
    cache = paged.PagedCache(ONE, ONE, dtype="float16", pages=4, page_size=16, kv_heads=2, hd=64, hd_v=32)
    assert cache.k_strides == (2048, 64, 128) and cache.v_strides == (1024, 32, 64)
    assert paged.PagedCache(ONE, ONE, dtype="float16", pages=4, page_size=16, kv_heads=2, hd=64, k_strides=[4096, 1024, 64]).k_strides == (4096, 1024, 64)
    with pytest.raises(NotImplementedError):
        paged.PagedCache(ONE, ONE, dtype="int8", pages=4, page_size=16, kv_heads=2, hd=64)
