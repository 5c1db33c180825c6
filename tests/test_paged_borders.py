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


# ---------------------------------------------------------------- what the binding is handed

class Tensor:
    """As much of a tensor as the binding looks at."""

    def __init__(self, dtype="bfloat16", numel=1 << 20, *, device=0, dense=True, ptr=4096, offset=0):
        self.dtype, self.ptr_, self.dense, self.at, self.shape, self.offset = f"torch.{dtype}", ptr, dense, device, (numel,), offset
        self.itemsize = {"bfloat16": 2, "float16": 2, "float32": 4, "int32": 4, "uint32": 4, "int64": 8, "float64": 8, "uint8": 1}[dtype]
        self.nbytes, self.device = numel * self.itemsize, f"cuda:{device}"

    def data_ptr(self):
        return self.ptr_

    def get_device(self):
        return self.at

    def is_contiguous(self):
        return self.dense

    def stride(self):
        return (1,) if self.dense else (2,)

    def untyped_storage(self):
        return type("Storage", (), {"nbytes": lambda _: self.nbytes + self.offset * self.itemsize})()

    def storage_offset(self):
        return self.offset


class Buffer:
    def __init__(self, nbytes, ptr=8192):
        self.nbytes, self.ptr = nbytes, ptr


@pytest.fixture
def calls(monkeypatch):
    """The library's part, which only writes down what it is called with."""
    from limn_b200 import paged

    seen = []

    class Library:
        def limn_b200_sdpa_paged_workspace(self, step, max_prefix, need):
            need._obj.value = 4096
            return 0

        limn_b200_kv_append = limn_b200_sdpa_paged = limn_b200_sdpa_paged_prefix = lambda self, *args: seen.append(args) or 0

    library = Library()
    monkeypatch.setattr(paged, "lib", lambda: library)
    return seen


EXTENTS = {"dtype": "bfloat16", "pages": 10, "page_size": 16, "kv_heads": 2, "hd": 64}  # 20480 elements a side


def batch(cache=None, **other):
    from limn_b200.paged import PagedBatch, PagedCache

    cache = cache or PagedCache(Tensor(), Tensor(), **EXTENTS)
    more = {"heads": 4, "batch": 3, "tokens": 5, "max_t_q": 2, "max_pages": 4, "page_table": Tensor("int32", 12), "q_start": Tensor("int32", 4), "kv_lens": Tensor("int32", 3),
            "workspace": Tensor("uint8", 4096)}
    return PagedBatch(cache, **{**more, **other})


@pytest.mark.parametrize("what, other", [
    ("bfloat16", {"k": Tensor("float16")}),
    ("bfloat16", {"v": Tensor("float32")}),
    ("GPU", {"k": Tensor(device=-1)}),
    ("reach", {"k": Tensor(numel=20479)}),
    ("reach", {"v": Buffer(2 * 20480 - 2)}),
    ("reach", {"k_strides": (4096, 64, 128), "k": Tensor(numel=20480)}),
    ("strides", {"k_strides": (2048, 64)}),
])
def test_pages_that_are_not_what_the_cache_says(what, other):
    from limn_b200.paged import PagedCache

    with pytest.raises(ValueError, match=what):
        PagedCache(**{"k": Tensor(), "v": Tensor(), **EXTENTS, **other})


def test_pages_of_a_shared_buffer():
    """A view shows fewer elements than its pages reach over: what counts is where its memory ends."""
    from limn_b200.paged import PagedCache

    shared = {**EXTENTS, "k_strides": (4096, 64, 128), "v_strides": (4096, 64, 128)}
    whole = Tensor(numel=9 * 4096 + 2048 + 2048)
    PagedCache(whole, Tensor(numel=9 * 4096 + 2048, offset=2048), **shared)
    PagedCache(whole.data_ptr(), Buffer(2 * (9 * 4096 + 2048)), **shared)
    with pytest.raises(ValueError, match="reach"):
        PagedCache(whole, Tensor(numel=9 * 4096 + 2047, offset=2048), **shared)


@pytest.mark.parametrize("what, other", [
    ("page_table", {"page_table": Tensor("int64", 12)}),
    ("page_table", {"page_table": Tensor("int32", 11)}),
    ("page_table", {"page_table": Tensor("int32", 12, dense=False)}),
    ("page_table", {"page_table": Buffer(47)}),
    ("q_start", {"q_start": Tensor("int32", 3)}),
    ("q_start", {"q_start": Tensor("int32", 4, device=-1)}),
    ("kv_lens", {"kv_lens": Tensor("int64", 3)}),
    ("kv_lens", {"kv_lens": Buffer(11)}),
    ("errors", {"errors": Tensor("int64", 1)}),
    ("one device", {"errors": Tensor("int32", 1, device=1)}),
    ("one device", {"workspace": Tensor("uint8", 4096, device=1)}),
    ("workspace", {"workspace": Tensor("uint8", 4095)}),
    ("workspace", {"workspace": Tensor("uint8", 4096, dense=False)}),
])
def test_arrays_that_a_batch_cannot_read(calls, what, other):
    batch()
    batch(page_table=Buffer(48), q_start=512, kv_lens=Buffer(12), errors=Tensor("uint32", 1), workspace=1 << 20)
    with pytest.raises(ValueError, match=what):
        batch(**other)


def test_a_workspace_that_only_says_it_is_on_the_cpu(calls):
    """Everything else is buffers, of which no device is known."""
    from limn_b200.paged import PagedCache

    with pytest.raises(ValueError, match="workspace"):
        batch(PagedCache(512, 512, **EXTENTS), page_table=512, q_start=512, kv_lens=512, workspace=Tensor("uint8", 4096, device=-1))


GOOD = {"q": Tensor(numel=5 * 4 * 64, ptr=16), "k": Tensor(numel=5 * 2 * 64, ptr=32), "v": Tensor(numel=5 * 2 * 64, ptr=48), "q_out": Tensor(numel=5 * 4 * 64, ptr=64),
        "frequencies": Tensor("float64", 32, ptr=80)}
BAD_FOR_APPEND = [
    ("q ", {"q": Tensor("float16", 1280)}), ("q ", {"q": Tensor(numel=1279)}), ("q ", {"q": Tensor(dense=False)}), ("q ", {"q": Tensor(device=1)}), ("q ", {"q": Tensor(device=-1)}),
    ("k ", {"k": Tensor(numel=639)}), ("v ", {"v": Tensor("float32")}), ("q_out", {"q_out": Tensor(dense=False)}), ("frequencies", {"frequencies": Tensor("float32", 32)}),
    ("frequencies", {"frequencies": Tensor("float64", 31)}), ("k ", {"k": Tensor("float32"), "k_strides": (512, 64)}), ("strides", {"k_strides": (512, 64, 1)}),
    ("strides", {"k_strides": (512, 64, 1), "v_strides": (512,)}),
]


@pytest.mark.parametrize("what, other", BAD_FOR_APPEND, ids=[f"{i}-{w}" for i, (w, _) in enumerate(BAD_FOR_APPEND)])
def test_operands_that_append_cannot_read(calls, what, other):
    step = batch()
    step.append(**GOOD, rotated=64)
    step.append(**{**GOOD, "k": Tensor(numel=1, dense=False, ptr=96)}, k_strides=(512, 64), rotated=64)  # with strides, a tensor says where it begins
    step.append(GOOD["k"], GOOD["v"])
    assert [call[1:5] for call in calls] == [(16, 32, 48, 64), (16, 96, 48, 64), (None, 32, 48, None)]
    with pytest.raises(ValueError, match=what):
        step.append(**{**GOOD, **other}, rotated=64)
    assert len(calls) == 3


@pytest.mark.parametrize("what, other", [
    ("q ", {"q": Tensor("float16", 1280)}), ("out", {"out": Tensor(numel=1279)}), ("out", {"out": Tensor(dense=False)}), ("lse", {"lse": Tensor("bfloat16", 20)}),
    ("lse", {"lse": Tensor("float32", 19)}), ("lse", {"lse": Tensor("float32", 20, device=1)}), ("strides", {"q_strides": (256, 64, 1), "out_strides": (256,)}),
])
def test_operands_that_attention_cannot_read(calls, what, other):
    step = batch()
    good = {"q": Tensor(numel=1280, ptr=16), "out": Tensor(numel=1280, ptr=32), "lse": Tensor("float32", 20, ptr=48)}
    table = Tensor("int32", 2, ptr=64)
    step.attention(**good)
    step.attention_with_prefix(**good, prefix_table=table, prefix_len=32)
    with pytest.raises(ValueError, match=what):
        step.attention(**{**good, **other})
    with pytest.raises(ValueError, match=what):
        step.attention_with_prefix(**{**good, **other}, prefix_table=table, prefix_len=32)
    for bad in (Tensor("int64", 2), Tensor("int32", 1), Tensor("int32", 2, dense=False)):
        with pytest.raises(ValueError, match="prefix_table"):
            step.attention_with_prefix(**good, prefix_table=bad, prefix_len=32)
    assert len(calls) == 2


def test_a_tensor_library():
    """torch's own tensors, here on the CPU, where no kernel could read them."""
    torch = pytest.importorskip("torch")
    from limn_b200.paged import PagedCache

    pages = torch.zeros(10, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        PagedCache(pages, pages, **EXTENTS)
    with pytest.raises(ValueError, match="bfloat16"):
        PagedCache(pages.float(), pages, **EXTENTS)
