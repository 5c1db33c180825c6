"""A paged key and value cache: new tokens into it, attention over it, attention behind a prefix that a batch shares.

    cache = PagedCache(k_pages, v_pages, dtype="bfloat16", pages=4096, page_size=16, kv_heads=8, hd=128)
    step = PagedBatch(cache, heads=32, batch=64, tokens=64, max_t_q=1, max_pages=512,
                      page_table=table, q_start=offsets, kv_lens=lengths)
    step.append(k, v, q=q, q_out=q, frequencies=freqs, rotated=128)
    step.attention(q, out, lse)

The binding of limn_b200_kv_append, limn_b200_sdpa_paged and limn_b200_sdpa_paged_prefix (include/limn_b200.h, which says
what each does with which extents). Every operand is device memory of the current device: an address, or an object
that carries one as `.ptr` (limn's buffers, limn_b200.runtime.DeviceBuffer) or `data_ptr()`. A tensor also says what it holds and where: one of another type or
device, one that is too small, or one that is not dense and comes without strides is refused with a ValueError. Offsets, lengths and tables are
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


# How an operand's address is read, by its type (asking an object for an attribute it lacks takes longer than all the rest of a call), and the types that
# say more of what they hold.
_ADDRESS_OF: dict[type, Callable[[Any], int | None]] = {type(None): lambda x: None, int: lambda x: x}
_TENSORS: set[type] = set()
_DTYPE_NAMES: dict[Any, str] = {}  # a tensor library's dtype objects


def _address(operand: Any) -> int | None:
    kind = type(operand)
    read = _ADDRESS_OF.get(kind)
    if read is None:
        read = attrgetter("ptr") if hasattr(operand, "ptr") else methodcaller("data_ptr")
        read(operand)  # raises before the type is remembered, where it has neither
        if not hasattr(operand, "ptr") and all(hasattr(operand, name) for name in ("dtype", "nbytes", "get_device", "is_contiguous")):
            _TENSORS.add(kind)
        _ADDRESS_OF[kind] = read
    return read(operand)


def _dtype_name(dtype: Any) -> str:
    name = _DTYPE_NAMES.get(dtype)
    if name is None:
        name = _DTYPE_NAMES[dtype] = str(dtype).rpartition(".")[2]
    return name


def _array(operand: Any, name: str, dtypes: tuple[str, ...], nbytes: int) -> tuple[int | None, int | None]:
    """Address and device of an array that a batch keeps, as far as it says: a dense tensor of one of `dtypes` (none: of any), or anything, of at least `nbytes`."""
    at = _address(operand)
    is_tensor = type(operand) in _TENSORS
    if is_tensor and ((dtypes and _dtype_name(operand.dtype) not in dtypes) or not operand.is_contiguous() or operand.get_device() < 0):
        raise ValueError(f"limn_b200: {name} must be a dense {' or '.join(dtypes)} tensor on a GPU, got {operand.dtype} on {operand.device}, strides {operand.stride()}")
    if getattr(operand, "nbytes", nbytes) < nbytes:
        raise ValueError(f"limn_b200: the {name} has {operand.nbytes} bytes, {nbytes} are needed")
    return at, operand.get_device() if is_tensor else None


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
        self._check("k", k, dtype, self.hd, self.k_strides)
        self._check("v", v, dtype, self.hd_v, self.v_strides)

    def _check(self, name: str, side: Any, dtype: str, width: int, strides: tuple[int, ...]) -> None:
        if len(strides) != 3:
            raise ValueError(f"limn_b200: the strides of {name} are (page, head, slot), got {strides}")
        _address(side)
        if type(side) in _TENSORS:
            if _dtype_name(side.dtype) != dtype or side.get_device() < 0:
                raise ValueError(f"limn_b200: the pages of {name} are {dtype} on a GPU, got {side.dtype} on {side.device}")
            room = side.untyped_storage().nbytes() // 2 - side.storage_offset()  # a view's pages may lie beyond what it shows of them
        elif hasattr(side, "nbytes"):
            room = side.nbytes // 2
        else:
            return
        reach = sum((n - 1) * stride for n, stride in zip((self.pages, self.kv_heads, self.page_size), strides, strict=True)) + width
        if reach > room and dtype in ("float16", "bfloat16"):  # (of other types the library serves none)
            raise ValueError(f"limn_b200: the pages of {name} reach over {reach} elements, there are {room}")


class PagedBatch:
    """A batch of sequences over a cache. `errors` is a device word that collects LIMN_B200_PAGED_BAD_* bits (the caller zeroes
    and reads it); `max_prefix` the longest shared prefix attention_with_prefix will be asked for, 0 for none (any other number takes the
    same room). `workspace` is 16-byte aligned device memory of at least what a batch of these extents has as `workspace_bytes`, such as the `workspace` of
    the batch over another layer of the same model, whose calls follow this one's on one stream; without one the batch allocates its own."""

    def __init__(self, cache: PagedCache, *, heads: int, batch: int, tokens: int, max_t_q: int, page_table: Any, max_pages: int,
                 q_start: Any, kv_lens: Any, first_position: int = 0, errors: Any = None, max_prefix: int = 1, workspace: Any = None):
        # the objects stay referenced as long as the step may read their memory
        self._held = (cache, page_table, q_start, kv_lens, errors)
        arrays = (_array(page_table, "page_table", ("int32",), 4 * batch * max_pages), _array(q_start, "q_start", ("int32",), 4 * (batch + 1)),
                  _array(kv_lens, "kv_lens", ("int32",), 4 * batch), _array(errors, "errors", ("int32", "uint32"), 4))
        self._step = Paged(_address(cache.k), _address(cache.v), *(at for at, _ in arrays),
                           (ctypes.c_longlong * 3)(*cache.k_strides), (ctypes.c_longlong * 3)(*cache.v_strides), cache.dtype, batch, heads,
                           cache.kv_heads, cache.hd, cache.hd_v, cache.page_size, cache.pages, max_pages, tokens, max_t_q, first_position)
        self._by_ref = ctypes.byref(self._step)
        self._step_at = ctypes.addressof(self._step)
        self._head_dim = cache.hd
        # (token, head) strides of dense operands: q, q_out, k, v and out
        self._dense = {"q": (heads * cache.hd, cache.hd), "k": (cache.kv_heads * cache.hd, cache.hd),
                       "v": (cache.kv_heads * cache.hd_v, cache.hd_v), "out": (heads * cache.hd_v, cache.hd_v)}
        self._packed: dict[tuple, tuple[Any, int]] = {}
        # what a tensor has to hold, if it is dense: type, bytes
        rows, kind = 2 * tokens, next(name for name, code in DTYPE_CODES.items() if code == cache.dtype)
        self._wants = {"q": (kind, rows * heads * cache.hd), "q_out": (kind, rows * heads * cache.hd), "k": (kind, rows * cache.kv_heads * cache.hd),
                       "v": (kind, rows * cache.kv_heads * cache.hd_v), "out": (kind, rows * heads * cache.hd_v), "lse": ("float32", 4 * tokens * heads)}
        loaded = lib()
        self._append, self._attend, self._attend_prefix = loaded.limn_b200_kv_append, loaded.limn_b200_sdpa_paged, loaded.limn_b200_sdpa_paged_prefix
        need = ctypes.c_ulonglong()
        check(lib().limn_b200_sdpa_paged_workspace(self._by_ref, max_prefix, ctypes.byref(need)), "sizing the workspace of a paged batch")
        self.workspace_bytes = need.value
        if workspace is None and need.value:
            workspace = DeviceBuffer(need.value)
        self.workspace = workspace
        self._workspace_at, device = _array(workspace, "workspace", (), need.value)
        devices = {device, *(device for _, device in arrays), *(x.get_device() for x in (cache.k, cache.v) if type(x) in _TENSORS)} - {None}
        if len(devices) > 1:
            raise ValueError(f"limn_b200: the arrays of a batch are on one device, got {sorted(devices)}")
        self._device = devices.pop() if devices else None

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
        at = self._at
        code = self._append(self._step_at, at(q, "q", q_strides), at(k, "k", k_strides), at(v, "v", v_strides), at(q_out, "q_out", q_out_strides), strides[1],
                            at(frequencies, "frequencies", None, ("float64", 4 * rotated)), rotated, PAIRING_CODES[pairing],
                            stream.handle if isinstance(stream, Stream) else stream)
        if code:
            check(code, "launching kv_append")

    def attention(self, q: Any, out: Any, lse: Any, *, q_strides=None, out_strides=None, causal: bool = True, scale: float | None = None,
                  stream: Any = None) -> None:
        """out = softmax(q k^T scale) v over each sequence's pages, lse its row statistic (tokens, heads) in float32. `scale`
        is hd ** -0.5 unless it is given."""
        strides = self._packed.get((q_strides, out_strides))
        if strides is None:
            strides = self._pack((q_strides, out_strides), ("q", "out"))
        at = self._at
        code = self._attend(self._step_at, at(q, "q", q_strides), at(out, "out", out_strides), at(lse, "lse"), strides[1], causal,
                            self._head_dim**-0.5 if scale is None else scale, self._workspace_at, self.workspace_bytes, stream.handle if isinstance(stream, Stream) else stream)
        if code:
            check(code, "launching sdpa_paged")
        _note_launch()

    def attention_with_prefix(self, q: Any, out: Any, lse: Any, *, prefix_table: Any, prefix_len: int, q_strides=None, out_strides=None,
                              causal: bool = True, scale: float | None = None, stream: Any = None) -> None:
        """The same with prefix_len keys of the pages prefix_table names in front of every sequence's own."""
        strides = self._packed.get((q_strides, out_strides))
        if strides is None:
            strides = self._pack((q_strides, out_strides), ("q", "out"))
        at, pages = self._at, -(-prefix_len // self._step.page_size)
        code = self._attend_prefix(self._step_at, at(q, "q", q_strides), at(out, "out", out_strides), at(lse, "lse"), strides[1],
                                   at(prefix_table, "prefix_table", None, ("int32", 4 * pages)), prefix_len, causal,
                                   self._head_dim**-0.5 if scale is None else scale, self._workspace_at, self.workspace_bytes,
                                   stream.handle if isinstance(stream, Stream) else stream)
        if code:
            check(code, "launching sdpa_paged_prefix")
        _note_launch()

    def _at(self, operand: Any, name: str, strides: tuple | None = None, wants: tuple[str, int] | None = None) -> int | None:
        """Where a call's operand begins; a tensor has the type and, without strides, the extent that the call goes by, and is on the batch's device."""
        if type(operand) not in _TENSORS:
            at = _address(operand)
            if type(operand) not in _TENSORS:  # (else seen for the first time)
                return at
        dtype, nbytes = wants or self._wants[name]
        # (one test of what nearly always holds, a tenth of a microsecond for each thing asked; why it does not is found out below)
        if (_DTYPE_NAMES.get(operand.dtype) == dtype and operand.get_device() == self._device
                and (strides is not None or (operand.nbytes >= nbytes and operand.is_contiguous()))):
            return operand.data_ptr()
        device = operand.get_device()
        if _dtype_name(operand.dtype) != dtype or device < 0 or (device != self._device and self._device is not None):
            where = "a GPU" if self._device is None else f"device {self._device}"
            raise ValueError(f"limn_b200: {name} must be {dtype} on {where}, got {operand.dtype} on {operand.device}")
        if strides is None and not (operand.is_contiguous() and operand.nbytes >= nbytes):
            raise ValueError(f"limn_b200: {name} without strides must be dense, of {nbytes} bytes, got shape {tuple(operand.shape)}, strides {operand.stride()}")
        return operand.data_ptr()

    def _pack(self, given: tuple, names: tuple[str, ...]):
        """The strides of a call as the library takes them; kept, since a batch's calls are alike step after step."""
        if any(strides is not None and len(strides) != 2 for strides in given):
            raise ValueError(f"limn_b200: strides are (token, head) pairs, got {given}")
        flat = [int(x) for strides, name in zip(given, names, strict=True) for x in (self._dense[name] if strides is None else strides)]
        if len(self._packed) >= 64:
            self._packed.clear()
        packed = (ctypes.c_longlong * len(flat))(*flat)
        self._packed[given] = packed, ctypes.addressof(packed)
        return self._packed[given]
