"""The paged cache and the rotary positions (include/itak_hip_kv.h): keys and values in pages of one storage, which sequences
name through tables, where a KvPool gives every slot rows of its own. No counterpart in the reference.

A serving program owns the pages: it decides which are free, which sequences share a prefix's, and hands every forward the
tables of the sequences in it (`PagedKv.set_batch`); then it goes through the layers.
"""
from __future__ import annotations

import ctypes as C
import math
from array import array
from typing import Optional, Sequence, Tuple

import numpy as np

from . import _native as N
from . import hip_compute
from .hip_compute import _check, _ptr, _raise_last

_ELEMS = {"f32": N.ELEM_F32, "f16": N.ELEM_F16, "bf16": N.ELEM_BF16}
_TORCH = {"torch.float32": N.ELEM_F32, "torch.float16": N.ELEM_F16, "torch.bfloat16": N.ELEM_BF16}
_SCALINGS = {"plain": N.ROTATION_PLAIN, "linear": N.ROTATION_LINEAR, "yarn": N.ROTATION_YARN}
_NAN = math.nan


def _filled(kind, *values):
    """The structure of these values; refused is an integer that its field would take modulo the field's size."""
    raw = kind(*values)
    for (name, _), value in zip(kind._fields_, values):
        if isinstance(value, int) and value != (getattr(raw, name) or 0):
            raise ValueError(f"{name}: {value} is out of range")
    return raw


class Rows:
    """A view of rows x heads x channels on the device (itak_rows): pointer, type, heads, strides in elements."""

    __slots__ = ("raw", "ref", "at", "rows", "channels", "keep")

    def __init__(self, ptr: int, elem: str, heads: int, row_stride: int = 0, head_stride: int = 0, keep=None, rows: int = -1,
                 channels: int = -1):
        if not 0 <= heads < 1 << 32:  # (a field would take it modulo its size; strides that far out are refused as they are)
            raise ValueError(f"heads: {heads} is out of range")
        self.raw = N.Rows(ptr, _ELEMS[elem] if isinstance(elem, str) else elem, heads, row_stride, head_stride)
        self.ref = C.byref(self.raw)
        self.at = C.addressof(self.raw)  # the view as the front module takes it
        self.rows, self.channels = rows, channels  # -1: of a pointer, as many as a call takes it for
        self.keep = keep  # what owns the memory

    @staticmethod
    def of(tensor) -> "Rows":
        """The view of a torch tensor [rows][heads][channels] on a GPU, whose channels lie side by side."""
        rows, heads, channels = tensor.shape
        if not tensor.is_cuda:
            raise ValueError("Rows.of: the tensor is not on a GPU")
        elem = _TORCH.get(str(tensor.dtype))
        if elem is None:
            raise ValueError(f"Rows.of: {tensor.dtype} is none of float32, float16, bfloat16")
        row_stride, head_stride, channel_stride = tensor.stride()
        if channels > 1 and channel_stride != 1:
            raise ValueError("Rows.of: the channels of a head do not lie side by side")
        if rows > 1 and heads > 1 and row_stride == 0 and head_stride == 0:  # (both zero stand for a dense view)
            raise ValueError("Rows.of: the tensor is one head's channels expanded to all rows and heads")
        # (A stride that is never taken may be anything; written out, a single row of a single head is not taken for dense.)
        return Rows(tensor.data_ptr(), elem, heads, row_stride if rows > 1 else heads * max(head_stride, channels),
                    head_stride if heads > 1 else channels, tensor, rows, channels)


def _holds(views: Sequence[Rows], rows: int, channels: int) -> None:
    for v in views:
        if v.rows >= 0 and (v.rows < rows or v.channels != channels):
            raise ValueError(f"a tensor of {v.rows} rows of {v.channels} channels where {rows} of {channels} are taken")


def _turning(rotation: Optional["Rotation"]) -> Optional[C.c_void_p]:
    if rotation is None:
        return None
    if not rotation._h:
        raise ValueError("the rotation is closed")
    return rotation._h


class Rotation:
    """Rotary positions (itak_rotation): `rotary_dim` channels of a head turn by position * frequency, pair by pair; adjacent
    pairs with `interleaved`, else half split. scaling "linear" divides the frequencies by `factor`, "yarn" only those of
    the pairs that turn seldom over `original_positions`. `amplitude` None: 1, of "yarn" 0.1 ln(factor) + 1."""

    def __init__(self, rotary_dim: int, *, base: float = 10000.0, interleaved: bool = False, scaling: str = "plain",
                 factor: float = 1.0, original_positions: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 amplitude: Optional[float] = None, device: int = 0):
        self._h = None
        self._hv = None  # the handle as the front module takes it
        self._lib = hip_compute._load()
        if scaling not in _SCALINGS:
            raise ValueError(f"scaling {scaling!r} is none of {', '.join(_SCALINGS)}")
        cfg = _filled(N.RotationConfig, base, rotary_dim, 1 if interleaved else 0, _SCALINGS[scaling], device, factor,
                      original_positions, beta_fast, beta_slow, amplitude or 0.0)
        handle = C.c_void_p()
        if self._lib.itak_rotation_create(C.byref(cfg), C.byref(handle)) != N.OK:
            _raise_last(None)
        self._h, self._hv = handle, handle.value
        self.rotary_dim = rotary_dim

    def close(self) -> None:
        if self._h:
            self._lib.itak_rotation_destroy(self._h)
            self._h = self._hv = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def frequencies(self) -> Tuple[np.ndarray, float]:
        """Radians a position of every pair, and what cosine and sine are multiplied by."""
        out, amplitude = np.empty(self.rotary_dim // 2), C.c_double()
        _check(None, self._lib.itak_rotation_frequencies(self._h, _ptr(out), C.byref(amplitude)))
        return out, amplitude.value

    def rotate_device(self, inputs: Sequence[Rows], outputs: Sequence[Rows], positions_ptr: int, rows: int, head_dim: int,
                      stream: int = 0, inverse: bool = False) -> None:
        """outputs[i] = inputs[i] turned by the rows' positions (int64 on the device), up to four tensors in one launch on
        `stream`; `inverse` turns back, which is what gradients of rotated rows go through."""
        status = hip_compute._front.rotate(self._hv, stream, head_dim, rows, positions_ptr, inputs, outputs, inverse)
        if status < 0:  # arguments that the front module leaves to ctypes
            n = len(inputs)
            if len(outputs) != n:
                raise ValueError("rotate_device: as many outputs as inputs")
            _holds((*inputs, *outputs), rows, head_dim)
            table = N.Rows * n
            status = self._lib.itak_rotate_device(_turning(self), stream, head_dim, rows, positions_ptr, table(*[r.raw for r in inputs]),
                                                  table(*[r.raw for r in outputs]), n, 1 if inverse else 0)
        if status:
            _raise_last(None)


class PageTables:
    """Page tables on the device (itak_page_tables), the caller's memory: of each sequence up to `stride` page ids and how many, and the
    free list."""

    __slots__ = ("raw", "ref", "at", "sequences", "free_words", "keep")

    def __init__(self, table_ptr: int, stride: int, pages_ptr: int, sequences: int, free_ptr: int = 0, free_count_ptr: int = 0, keep=None):
        self.raw = _filled(N.PageTables, table_ptr or None, stride, pages_ptr or None, free_ptr or None, free_count_ptr or None, sequences, 0)
        self.ref = C.byref(self.raw)
        self.at = C.addressof(self.raw)  # as the front module takes it
        self.sequences = sequences
        self.free_words = None  # of the free list, where that is known
        self.keep = keep  # what owns the memory

    @staticmethod
    def of(table, pages, free=None, free_count=None) -> "PageTables":
        """Of int32 tensors on a GPU: table [sequences][stride], pages [sequences], free [page_count], free_count [1]."""
        for name, t, dims in (("table", table, 2), ("pages", pages, 1), ("free", free, 1), ("free_count", free_count, 1)):
            if t is not None and not (t.is_cuda and str(t.dtype) == "torch.int32" and t.dim() == dims and t.is_contiguous()):
                raise ValueError(f"PageTables.of: {name} is no dense int32 tensor of {dims} dimensions on a GPU")
            if t is not None and t.device != table.device:
                raise ValueError(f"PageTables.of: {name} is on another device than table")
        if pages.shape[0] != table.shape[0]:
            raise ValueError(f"PageTables.of: pages of {pages.shape[0]} sequences, tables of {table.shape[0]}")
        if free_count is not None and free_count.shape[0] != 1:
            raise ValueError(f"PageTables.of: free_count of {free_count.shape[0]} words")
        tables = PageTables(table.data_ptr(), table.shape[1], pages.data_ptr(), table.shape[0], 0 if free is None else free.data_ptr(),
                            0 if free_count is None else free_count.data_ptr(), (table, pages, free, free_count))
        tables.free_words = None if free is None else free.shape[0]
        return tables


def _words(values, kind: str, low: int, high: int, what: str):
    """Host values as an array of 32-bit words; its address and count."""
    if isinstance(values, np.ndarray):
        if values.dtype.kind not in "iu" or values.ndim != 1:
            raise ValueError(f"{what} are no integers in a row")
        if values.size and (values.min() < low or values.max() > high):
            raise ValueError(f"{what} beyond {low} .. {high}")
        words = np.ascontiguousarray(values, dtype=np.int32 if kind == "i" else np.uint32)
        return words, _ptr(words) if words.size else None, words.size
    words = array(kind)
    try:
        words.extend(values)
    except OverflowError:
        raise ValueError(f"{what} beyond {low} .. {high}") from None
    ptr, count = words.buffer_info()
    return words, ptr if count else None, count


class PagedKv:
    """Keys and values in pages (itak_paged): storage [layer][page][side][kv_head][page row][channel], side 0 = keys. The storage
    is the caller's (`storage_ptr`, `storage_bytes`: at least `PagedKv.bytes_for(...)`) or the cache's own."""

    def __init__(self, layers: int, num_kv_heads: int, head_dim: int, *, elem: str = "f16", page_rows: int = 64,
                 page_count: int, max_sequences: int = 64, max_table_pages: int = 0, device: int = 0, storage_ptr: int = 0,
                 storage_bytes: int = 0):
        self._h = None
        self._hv = 0  # the handle as the front module takes it
        self._lib = hip_compute._load()
        cfg = self._config(layers, num_kv_heads, head_dim, elem, page_rows, page_count, max_sequences, max_table_pages, device,
                           storage_ptr, storage_bytes)
        handle = C.c_void_p()
        if self._lib.itak_paged_create(C.byref(cfg), C.byref(handle)) != N.OK:
            _raise_last(None)
        self._h, self._hv = handle, handle.value
        self.page_rows = page_rows
        self.page_count = page_count
        self.head_dim = head_dim
        self._rows = 0  # of the batch

    @staticmethod
    def _config(layers, num_kv_heads, head_dim, elem, page_rows, page_count, max_sequences=1, max_table_pages=0, device=0,
                storage_ptr=0, storage_bytes=0):
        return _filled(N.PagedConfig, layers, _ELEMS[elem], num_kv_heads, head_dim, page_count, page_rows, max_sequences,
                       max_table_pages, device, 0, storage_ptr or None, storage_bytes)

    @staticmethod
    def bytes_for(layers: int, num_kv_heads: int, head_dim: int, *, elem: str = "f16", page_rows: int = 64,
                  page_count: int) -> int:
        """Bytes of storage such a cache needs."""
        cfg = PagedKv._config(layers, num_kv_heads, head_dim, elem, page_rows, page_count)
        return int(N.load().itak_paged_storage_bytes(C.byref(cfg)))

    def _done(self, status: int) -> None:
        if status != N.OK:
            if not self._h:
                raise ValueError("the paged cache is closed")
            _raise_last(self._h, lib_error=(self._lib.itak_paged_last_error, self._lib.itak_paged_last_error_info))

    def close(self) -> None:
        if self._h:
            self._lib.itak_paged_destroy(self._h)
            self._h, self._hv = None, 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_stream(self, stream_handle: int) -> None:
        self._done(self._lib.itak_paged_set_stream(self._h, stream_handle))

    def synchronize(self) -> None:
        self._done(self._lib.itak_paged_synchronize(self._h))

    def storage_ptr(self) -> int:
        return int(self._lib.itak_paged_storage(self._h) or 0)

    def enable_trees(self, most_rows: int) -> None:
        """Lets batches be trees, of up to `most_rows` new rows in all (itak_paged_enable_trees); once."""
        if not 0 <= most_rows < 1 << 64:
            raise ValueError(f"most_rows: {most_rows} is out of range")
        self._done(self._lib.itak_paged_enable_trees(self._h, most_rows))

    def set_batch(self, items: Sequence[Tuple[int, int]], pages: Sequence[Sequence[int]],
                  parents: Optional[Sequence[int]] = None) -> None:
        """The sequences of the next forward: (positions held, new rows) of each, and its page ids in order. `parents` makes the new
        rows trees: of all rows in order the number of the row of the same sequence that it continues, or -1."""
        front = hip_compute._front
        status = front.set_batch(self._hv, items, pages) if parents is None else front.set_batch_tree(self._hv, items, pages, parents)
        if status >= 0:
            self._done(status)
            self._rows = sum([rows for _, rows in items])
            return
        n = len(items)
        if len(pages) != n:
            raise ValueError("set_batch: one table of pages a sequence")
        raw = (N.PagedItem * n)()
        for at, (position, rows), table in zip(raw, items, pages):
            if not (0 <= position < 1 << 64 and 0 <= rows < 1 << 32):  # (a field would take them modulo its size)
                raise ValueError(f"set_batch: ({position}, {rows}) is no position and rows")
            at.position, at.rows, at.pages = position, rows, len(table)
        if n and isinstance(pages[0], np.ndarray):
            ids = np.concatenate(pages)
            if ids.size and (ids.dtype.kind not in "iu" or ids.min() < 0 or ids.max() > 0xFFFFFFFF):
                raise ValueError("set_batch: page ids are integers of 32 bits")
            ids = np.ascontiguousarray(ids, dtype=np.uint32)
            ptr, count = _ptr(ids), ids.size
        else:
            ids = array("I")
            for table in pages:
                ids.extend(table)
            ptr, count = ids.buffer_info()
        all_rows = sum(int(rows) for _, rows in items)
        if parents is None:
            self._done(self._lib.itak_paged_set_batch(self._h, raw, n, ptr if count else None, count))
        else:
            words, parents_ptr, named = _words(parents, "i", -(1 << 31), (1 << 31) - 1, "parents")
            if named != all_rows:
                raise ValueError(f"set_batch: {named} parents of {all_rows} new rows")
            if parents_ptr is None:
                parents_ptr = C.addressof(C.c_int32())  # (of no rows: not read)
            self._done(self._lib.itak_paged_set_batch_tree(self._h, raw, n, ptr if count else None, count, parents_ptr))
        self._rows = all_rows

    def fit_tables_device(self, tables: PageTables, lengths_ptr: int, rows: Optional[Sequence[int]] = None, status_ptr: int = 0) -> None:
        """Page tables to lengths on the device (int32 [sequences]), and `rows` new rows on top of each: pages from the free list, or back."""
        if tables.free_words is not None and tables.free_words < self.page_count:
            raise ValueError(f"a free list of {tables.free_words} words for {self.page_count} pages")
        status = hip_compute._front.fit_tables(self._hv, tables.at, tables.sequences, lengths_ptr, rows, status_ptr)
        if status >= 0:
            self._done(status)
            return
        words, rows_ptr, named = _words(rows, "I", 0, (1 << 32) - 1, "rows") if rows is not None else (None, None, tables.sequences)
        if named != tables.sequences:
            raise ValueError(f"rows of {named} sequences, tables of {tables.sequences}")
        self._done(self._lib.itak_paged_fit_tables_device(self._h, tables.ref, lengths_ptr or None, rows_ptr, status_ptr or None))

    def set_batch_device(self, tables: PageTables, positions_ptr: int, rows: Sequence[int], most_positions: int, parents_ptr: int = 0,
                         status_ptr: int = 0) -> None:
        """The batch from positions (int32 [sequences]), tables and parents (int32 [sum rows]) on the device; `rows` new rows of each sequence,
        behind at most `most_positions`."""
        done = hip_compute._front.set_batch_device(self._hv, tables.at, tables.sequences, positions_ptr, rows, most_positions, parents_ptr,
                                                   status_ptr)
        if done >= 0:
            self._done(done >> 32)
            self._rows = done & 0xFFFFFFFF
            return
        words, rows_ptr, named = _words(rows, "I", 0, (1 << 32) - 1, "rows")
        if named != tables.sequences:
            raise ValueError(f"rows of {named} sequences, tables of {tables.sequences}")
        if not 0 <= most_positions < 1 << 64:
            raise ValueError(f"most_positions: {most_positions} is out of range")
        self._done(self._lib.itak_paged_set_batch_device(self._h, tables.ref, positions_ptr or None, rows_ptr, most_positions,
                                                         parents_ptr or None, status_ptr or None))
        self._rows = sum(words.tolist())

    def batch_rows_device(self, positions_ptr: int = 0, slots_ptr: int = 0) -> None:
        """Every row's position in the text and its row of the storage (page * page_rows + row): int64 [rows] each; -1 of rows left out."""
        status = hip_compute._front.batch_rows(self._hv, positions_ptr, slots_ptr)
        self._done(status if status >= 0 else self._lib.itak_paged_batch_rows_device(self._h, positions_ptr or None, slots_ptr or None))

    def accept_device(self, tokens_ptr: int, chosen_ptr: int, path_ptr: int, next_ptr: int) -> None:
        """The walk down every tree along the tokens chosen: `path` [rows] its row numbers and then -1, `next` [sequences] the choice at its
        end (int32 all)."""
        status = hip_compute._front.accept(self._hv, tokens_ptr, chosen_ptr, path_ptr, next_ptr)
        self._done(status if status >= 0 else self._lib.itak_paged_accept_device(self._h, tokens_ptr or None, chosen_ptr or None,
                                                                                 path_ptr or None, next_ptr or None))

    def keep_device(self, path_ptr: int, lengths_ptr: int = 0) -> None:
        """The rows of every path to the sequence's next positions, on all layers; `lengths` [sequences] the positions held then."""
        status = hip_compute._front.keep(self._hv, path_ptr, lengths_ptr)
        self._done(status if status >= 0 else self._lib.itak_paged_keep_device(self._h, path_ptr or None, lengths_ptr or None))

    def append_device(self, layer: int, k: Rows, v: Rows, rotation: Optional[Rotation] = None) -> None:
        """The batch's new rows into their pages, keys turned by their positions if `rotation` is given."""
        status = hip_compute._front.append(self._hv, self._rows, self.head_dim, layer, k, v,
                                           0 if rotation is None else rotation._hv)
        if status < 0:
            _holds((k, v), self._rows, self.head_dim)
            status = self._lib.itak_paged_append_device(self._h, layer, k.ref, v.ref, _turning(rotation))
        if status:
            self._done(status)

    def attention_device(self, layer: int, q: Rows, out: Rows, *, scale: Optional[float] = None, softcap: float = 0.0,
                         window: int = 0, rotation: Optional[Rotation] = None) -> None:
        """Attention of the batch's new positions over pages that hold their rows already."""
        status = hip_compute._front.paged_attention(self._hv, self._rows, self.head_dim, layer, q, out, scale, softcap, window,
                                                    0 if rotation is None else rotation._hv)
        if status < 0:
            _holds((q, out), self._rows, self.head_dim)
            status = self._lib.itak_paged_attention_device(self._h, layer, q.ref, out.ref, _NAN if scale is None else scale, softcap,
                                                           window, _turning(rotation))
        if status:
            self._done(status)

    def attention_step_device(self, layer: int, q: Rows, k: Rows, v: Rows, out: Rows, *, scale: Optional[float] = None,
                              softcap: float = 0.0, window: int = 0, rotation: Optional[Rotation] = None) -> None:
        """Append the batch's new rows, then attend; queries and keys turned first if `rotation` is given."""
        status = hip_compute._front.paged_step(self._hv, self._rows, self.head_dim, layer, q, k, v, out, scale, softcap, window,
                                               0 if rotation is None else rotation._hv)
        if status < 0:
            _holds((q, k, v, out), self._rows, self.head_dim)
            status = self._lib.itak_paged_step_device(self._h, layer, q.ref, k.ref, v.ref, out.ref, _NAN if scale is None else scale,
                                                      softcap, window, _turning(rotation))
        if status:
            self._done(status)
