"""A paged key and value cache: new tokens into it, attention over it, attention behind a prefix that a batch shares.

    cache = PagedCache(k_pages, v_pages, dtype="bfloat16", pages=4096, page_size=16, kv_heads=8, hd=128)
    step = PagedBatch(cache, heads=32, batch=64, tokens=64, max_t_q=1, max_pages=512,
                      page_table=table, q_start=offsets, kv_lens=lengths)
    step.append(k, v, q=q, q_out=q, frequencies=freqs, rotated=128)
    step.attention(q, out, lse)

The binding of limn_b200_kv_append, limn_b200_sdpa_paged and limn_b200_sdpa_paged_prefix (include/limn_b200.h, which says
what each does with which extents). Every operand is device memory of the current device: an address, or an object
that carries one as `.ptr` (limn's buffers, limn_b200.runtime.DeviceBuffer) or `data_ptr()`. Offsets, lengths and tables are
int32 and are read on the device by each call, so one PagedBatch serves step after step, and its captured calls follow what
the arrays hold when they are replayed. Calls launch on `stream` (None: the legacy default stream), do not synchronise and
allocate nothing; a PagedBatch allocates its workspace when it is made, unless it is given one. Calls of one PagedBatch
that can overlap on the GPU would share that workspace: give each stream a PagedBatch of its own. Captured calls keep using it:
keep the PagedBatch as long as the graph.
"""

from __future__ import annotations

import ctypes
from collections.abc import Callable
from operator import attrgetter, methodcaller
from typing import Any

from limn_b200._lib import DTYPE_CODES, PAIRING_CODES, Paged, check, lib
from limn_b200.registry import _note_launch
from limn_b200.runtime import DeviceBuffer, Stream


# How an operand's address is read, by its type (asking an object for an attribute it lacks takes longer than all the rest of a call).
_ADDRESS_OF: dict[type, Callable[[Any], int | None]] = {type(None): lambda x: None, int: lambda x: x}


def _address(operand: Any) -> int | None:
    kind = type(operand)
    read = _ADDRESS_OF.get(kind)
    if read is None:
        read = attrgetter("ptr") if hasattr(operand, "ptr") else methodcaller("data_ptr")
        read(operand)  # raises before the type is remembered, where it has neither
        _ADDRESS_OF[kind] = read
    return read(operand)


class PagedCache:
    """The pages of one layer's keys and values. Strides are (page, head, slot) in elements; without them the pages are
    dense, (pages, page_size, kv_heads, width)."""

    def __init__(self, k: Any, v: Any, *, dtype: str, pages: int, page_size: int, kv_heads: int, hd: int, hd_v: int | None = None,
                 k_strides=None, v_strides=None):
        if dtype not in DTYPE_CODES:
            raise NotImplementedError(f"limn_b200: a paged cache has no kernel for dtype {dtype}")
        self.k, self.v = k, v
        self.dtype = DTYPE_CODES[dtype]
        self.pages, self.page_size, self.kv_heads = pages, page_size, kv_heads
        self.hd, self.hd_v = hd, hd if hd_v is None else hd_v
        self.k_strides = tuple(k_strides or (page_size * kv_heads * self.hd, self.hd, kv_heads * self.hd))
        self.v_strides = tuple(v_strides or (page_size * kv_heads * self.hd_v, self.hd_v, kv_heads * self.hd_v))


class PagedBatch:
    """A batch of sequences over a cache. `errors` is a device word that collects LIMN_B200_PAGED_BAD_* bits (the caller zeroes
    and reads it); `max_prefix` the longest shared prefix attention_with_prefix will be asked for, 0 for none (any other number takes the
    same room). `workspace` is 16-byte aligned device memory of at least what a batch of these extents has as `workspace_bytes`, such as the `workspace` of
    the batch over another layer of the same model, whose calls follow this one's on one stream; without one the batch allocates its own."""

    def __init__(self, cache: PagedCache, *, heads: int, batch: int, tokens: int, max_t_q: int, page_table: Any, max_pages: int,
                 q_start: Any, kv_lens: Any, first_position: int = 0, errors: Any = None, max_prefix: int = 1, workspace: Any = None):
        # the objects stay referenced as long as the step may read their memory
        self._held = (cache, page_table, q_start, kv_lens, errors)
        self._step = Paged(_address(cache.k), _address(cache.v), _address(page_table), _address(q_start), _address(kv_lens), _address(errors),
                           (ctypes.c_longlong * 3)(*cache.k_strides), (ctypes.c_longlong * 3)(*cache.v_strides), cache.dtype, batch, heads,
                           cache.kv_heads, cache.hd, cache.hd_v, cache.page_size, cache.pages, max_pages, tokens, max_t_q, first_position)
        self._by_ref = ctypes.byref(self._step)
        self._head_dim = cache.hd
        # (token, head) strides of dense operands: q, q_out, k, v and out
        self._dense = {"q": (heads * cache.hd, cache.hd), "k": (cache.kv_heads * cache.hd, cache.hd),
                       "v": (cache.kv_heads * cache.hd_v, cache.hd_v), "out": (heads * cache.hd_v, cache.hd_v)}
        self._packed: dict[tuple, Any] = {}
        loaded = lib()
        self._append, self._attend, self._attend_prefix = loaded.limn_b200_kv_append, loaded.limn_b200_sdpa_paged, loaded.limn_b200_sdpa_paged_prefix
        need = ctypes.c_ulonglong()
        check(lib().limn_b200_sdpa_paged_workspace(self._by_ref, max_prefix, ctypes.byref(need)), "sizing the workspace of a paged batch")
        self.workspace_bytes = need.value
        if workspace is None and need.value:
            workspace = DeviceBuffer(need.value)
        if getattr(workspace, "nbytes", need.value) < need.value:
            raise ValueError(f"limn_b200: the workspace has {workspace.nbytes} bytes, {need.value} are needed")
        self.workspace = workspace
        self._workspace_at = _address(workspace)

    def append(self, k: Any, v: Any, *, q: Any = None, q_out: Any = None, k_strides=None, v_strides=None, q_strides=None, q_out_strides=None,
               frequencies: Any = None, rotated: int = 0, pairing: str = "halves", stream: Any = None) -> None:
        """Keys and values of the step's tokens into their slots, turned to their positions; q turned into q_out beside them.
        Strides are (token, head) tuples in
        elements; without them an operand is dense, (tokens, heads, width)."""
        if pairing not in PAIRING_CODES:
            raise ValueError(f"limn_b200: kv_append knows the pairings {sorted(PAIRING_CODES)}, not {pairing!r}")
        strides = self._packed.get((q_strides, q_out_strides, k_strides, v_strides))
        if strides is None:
            strides = self._pack((q_strides, q_out_strides, k_strides, v_strides), ("q", "q", "k", "v"))
        code = self._append(self._by_ref, _address(q), _address(k), _address(v), _address(q_out), strides, _address(frequencies), rotated,
                            PAIRING_CODES[pairing], stream.handle if isinstance(stream, Stream) else stream)
        if code:
            check(code, "launching kv_append")

    def attention(self, q: Any, out: Any, lse: Any, *, q_strides=None, out_strides=None, causal: bool = True, scale: float | None = None,
                  stream: Any = None) -> None:
        """out = softmax(q k^T scale) v over each sequence's pages, lse its row statistic (tokens, heads) in float32. `scale`
        is hd ** -0.5 unless it is given."""
        strides = self._packed.get((q_strides, out_strides))
        if strides is None:
            strides = self._pack((q_strides, out_strides), ("q", "out"))
        code = self._attend(self._by_ref, _address(q), _address(out), _address(lse), strides, causal, self._head_dim**-0.5 if scale is None else scale,
                            self._workspace_at, self.workspace_bytes, stream.handle if isinstance(stream, Stream) else stream)
        if code:
            check(code, "launching sdpa_paged")
        _note_launch()

    def attention_with_prefix(self, q: Any, out: Any, lse: Any, *, prefix_table: Any, prefix_len: int, q_strides=None, out_strides=None,
                              causal: bool = True, scale: float | None = None, stream: Any = None) -> None:
        """The same with prefix_len keys of the pages prefix_table names in front of every sequence's own."""
        strides = self._packed.get((q_strides, out_strides))
        if strides is None:
            strides = self._pack((q_strides, out_strides), ("q", "out"))
        code = self._attend_prefix(self._by_ref, _address(q), _address(out), _address(lse), strides, _address(prefix_table), prefix_len, causal,
                                   self._head_dim**-0.5 if scale is None else scale, self._workspace_at, self.workspace_bytes,
                                   stream.handle if isinstance(stream, Stream) else stream)
        if code:
            check(code, "launching sdpa_paged_prefix")
        _note_launch()

    def _pack(self, given: tuple, names: tuple[str, ...]):
        """The strides of a call as the library takes them; kept, since a batch's calls are alike step after step."""
        flat = [int(x) for strides, name in zip(given, names, strict=True) for x in (self._dense[name] if strides is None else strides)]
        if len(flat) != 2 * len(names):
            raise ValueError(f"limn_b200: strides are (token, head) pairs, got {given}")
        if len(self._packed) >= 64:
            self._packed.clear()
        packed = self._packed[given] = (ctypes.c_longlong * len(flat))(*flat)
        return packed
