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

    def set_batch(self, items: Sequence[Tuple[int, int]], pages: Sequence[Sequence[int]]) -> None:
        """The sequences of the next forward: (positions held, new rows) of each, and its page ids in order."""
        status = hip_compute._front.set_batch(self._hv, items, pages)
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
        self._done(self._lib.itak_paged_set_batch(self._h, raw, n, ptr if count else None, count))
        self._rows = sum(int(rows) for _, rows in items)

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
