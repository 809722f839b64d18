"""Operators of a decoder layer on torch tensors in device memory, around a K/V cache in pages.

``Rope`` rotates queries and keys; ``PagedCache`` is one layer's cache, whose
pages, page tables and lengths belong to the caller; ``PagedBatch`` is what a
step's sequences look like. They serve and give no gradients: tensors that
require one are refused outside torch.no_grad(). Every call enqueues its kernels on torch's current
stream of the cache's device and returns without waiting. It can be captured
into a graph, and replayed with other contents of the same tensors.
"""
from __future__ import annotations

import ctypes
import sys

from . import _capi
from ._capi import check, library

__all__ = ["Rope", "PagedCache", "PagedBatch"]

_TYPES = {"torch.float32": 1, "torch.float16": 2, "torch.bfloat16": 3}
_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
_codes: dict = {}  # torch dtype -> jfh_value_type


def _type(x, name: str) -> int:
    t = _codes.get(x.dtype)
    if t is None:
        t = _TYPES.get(str(x.dtype))
        if t is None:
            raise ValueError(f"{name} holds {x.dtype}: float32, float16 and bfloat16 are supported")
        _codes[x.dtype] = t
    return t


def _count(v: int, name: str) -> int:
    """A number for a C uint32_t, which ctypes would cut to its low 32 bits."""
    if not 0 <= v <= 0xFFFFFFFF:
        raise _capi.InvalidArgument(1, f"{name} must be 0 to 2^32 - 1, not {v}")
    return v


def _no_gradient(name: str) -> None:
    """Of a tensor that requires one."""
    if _torch().is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and these operators give none: call them under torch.no_grad()")


def _rows(x, name: str, device: int) -> _capi.Rows:
    """A tensor [rows, heads, head dim] of any strides whose heads are contiguous."""
    shape, stride = x.shape, x.stride()
    if x.requires_grad:
        _no_gradient(name)
    if len(shape) != 3:
        raise ValueError(f"{name} must be [rows, heads, head dim]")
    if x.get_device() != device or device < 0:
        raise ValueError(f"{name} must be on GPU {device}")
    if stride[2] != 1 and shape[2] > 1:
        raise ValueError(f"the values of a head of {name} must be contiguous")
    return _capi.Rows(x.data_ptr(), stride[0], stride[1], shape[0], shape[1], shape[2], _type(x, name))


def _array(x, name: str, dtype: str, device: int, shape: tuple | None = None) -> int:
    """Address of a contiguous device array."""
    if x.dtype is not getattr(_torch(), dtype) or x.get_device() != device or device < 0 or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor on GPU {device}")
    if shape is not None and x.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}, not {list(x.shape)}")
    if x.requires_grad:
        _no_gradient(name)
    return x.data_ptr()


def _torch():
    return sys.modules["torch"]  # there once the caller has a tensor


_current = None  # device -> address of torch's current stream


def _stream(device: int) -> int:
    global _current
    if _current is None:
        # without the Stream object around it, which takes longer than the rest of a small call's checks
        _current = getattr(_torch()._C, "_cuda_getCurrentRawStream", None) or (
            lambda d: _torch().cuda.current_stream(d).cuda_stream)
    return _current(device)


def _kept(i: int, doc: str) -> property:
    """A tensor whose address a handle has passed on: read-only, since another one would leave the address behind."""
    return property(lambda self: self._tensors[i], doc=doc)


class Rope:
    """Rotary positions (jfh_rope_params): the leading n_rot values of a head turn in pairs,
    (i, i + n_rot / 2) in the "half" layout, (2 i, 2 i + 1) in the "interleaved" one, by position *
    base^(-2 i / n_rot); ``scaling`` "linear", "ntk" or "yarn" stretches the angles for contexts
    ``factor`` times the trained one."""

    def __init__(self, n_rot: int, base: float = 1.0e6, layout: str = "half", scaling: str = "none", factor: float = 1.0,
                 original_context: int = 32768, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 attention_factor: float = 0.0):
        self._h = ctypes.c_void_p()
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}")
        if scaling not in _SCALINGS:
            raise ValueError(f"scaling must be one of {sorted(_SCALINGS)}")
        params = _capi.RopeParams(_count(n_rot, "n_rot"), _LAYOUTS[layout], _SCALINGS[scaling],
                                  _count(original_context, "original_context"), base, factor, beta_fast, beta_slow,
                                  attention_factor)
        check(library().jfh_rope_create(ctypes.byref(params), ctypes.byref(self._h)))

    def close(self) -> None:
        if self._h:
            library().jfh_rope_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def handle(self) -> ctypes.c_void_p:
        if not self._h:  # a null handle would be a call without rotation
            raise _capi.InvalidArgument(1, "the rotation is closed")
        return self._h

    def rotate(self, x, positions, out=None):
        """x [rows, heads, head dim] rotated by positions (int32 [rows]) into out, which may be x or
        have another type; a new tensor like x by default. Returns out."""
        if out is None:
            out = _torch().empty_like(x)
        device = x.get_device()
        a, b = _rows(x, "x", device), _rows(out, "out", device)
        at = _array(positions, "positions", "int32", device, (x.shape[0],))
        check(library().jfh_rope_rotate(self._h, ctypes.byref(a), at, ctypes.byref(b), device, _stream(device)))
        return out


class PagedBatch:
    """The sequences of a step (jfh_paged_batch), int32 tensors on the cache's GPU: table [sequences,
    pages], lengths [sequences] (slots in use, the new rows included) and row_starts [sequences + 1].
    max_rows and max_length bound the rows of a sequence and its length. The tensors' contents may change
    between calls, the tensors and their storage may not."""

    table = _kept(0, "int32 [sequences, pages]")
    lengths = _kept(1, "int32 [sequences]")
    row_starts = _kept(2, "int32 [sequences + 1]")
    device = property(lambda self: self._device, doc="ordinal of the GPU")

    def __init__(self, table, lengths, row_starts, max_rows: int, max_length: int):
        device = table.get_device()
        if table.dim() != 2:
            raise ValueError("table must be [sequences, pages]")
        n = table.shape[0]
        self._tensors = (table, lengths, row_starts)
        self._device = device
        self.c = _capi.PagedBatch(_array(table, "table", "int32", device),
                                  _array(lengths, "lengths", "int32", device, (n,)),
                                  _array(row_starts, "row_starts", "int32", device, (n + 1,)), n, table.shape[1],
                                  _count(max_rows, "max_rows"), _count(max_length, "max_length"))
        self.workspaces: dict = {}
        self.ref = ctypes.byref(self.c)


class PagedCache:
    """One layer's K/V cache in pages (jfh_paged_cache): k and v [pages, K/V heads, page size, head
    dim], float16 or bfloat16, of equal strides (a permuted view of another order will do); weights
    (float32) and positions (int32) [pages, K/V heads, page size], which only a cache that is cut needs. The
    tensors' contents may change between calls, the tensors and their storage may not."""

    k = _kept(0, "[pages, K/V heads, page size, head dim]")
    v = _kept(1, "like k")
    weights = _kept(2, "float32 [pages, K/V heads, page size] or None")
    positions = _kept(3, "int32 [pages, K/V heads, page size] or None")
    device = property(lambda self: self._device, doc="ordinal of the GPU")

    def __init__(self, k, v, weights=None, positions=None):
        device = k.get_device()
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError("k and v must be [pages, K/V heads, page size, head dim] of one type and equal strides")
        if not k.is_cuda or v.get_device() != device:
            raise ValueError("k and v must be on one GPU")
        if k.stride(3) != 1:
            raise ValueError("the values of a head must be contiguous")
        for x, name in ((k, "k"), (v, "v")):
            if x.requires_grad:
                _no_gradient(name)
        pages, heads, page_size, dim = k.shape
        meta = (pages, heads, page_size)
        self._tensors = (k, v, weights, positions)
        self._device = device
        self.c = _capi.PagedCache(
            k.data_ptr(), v.data_ptr(),
            None if weights is None else _array(weights, "weights", "float32", device, meta),
            None if positions is None else _array(positions, "positions", "int32", device, meta),
            k.stride(0), k.stride(1), k.stride(2), pages, page_size, heads, dim, _type(k, "k"), device)
        self.ref = ctypes.byref(self.c)
        self.shape = (heads, dim, page_size)

    def _of(self, batch: PagedBatch):
        if batch._device != self._device:
            raise ValueError(f"the batch is on GPU {batch._device}, the cache on GPU {self._device}")
        return batch.ref

    def _workspace(self, batch: PagedBatch, call: str, *args):
        """Address and size of a call's workspace (and the tensor that holds it), from torch's allocator:
        ordered by the current stream, and a captured graph's own. Its size goes by the shapes alone."""
        key = (call, self.shape, *((a.n_rows, a.n_head) if isinstance(a, _capi.Rows) else a for a in args))
        size = batch.workspaces.get(key)
        if size is None:
            need = ctypes.c_size_t()
            check(getattr(library(), f"jfh_paged_{call}_workspace")(
                self.ref, batch.ref, *(ctypes.byref(a) if isinstance(a, _capi.Rows) else a for a in args), ctypes.byref(need)))
            size = batch.workspaces[key] = need.value
        if size == 0:
            return None, 0, None
        space = _torch().empty(size, dtype=_torch().uint8, device=self._tensors[0].device)
        return space.data_ptr(), size, space

    def append(self, batch: PagedBatch, k, v, positions=None, rope: Rope | None = None) -> None:
        """Writes a step's rows k and v [rows, K/V heads, head dim] at its sequences' last slots, k
        rotated by rope; positions int32 [rows]."""
        a, b = _rows(k, "k", self._device), _rows(v, "v", self._device)
        at = None if positions is None else _array(positions, "positions", "int32", self._device, (k.shape[0],))
        check(library().jfh_paged_append(self.ref, self._of(batch), ctypes.byref(a), ctypes.byref(b),
                                         None if rope is None else rope.handle, at, _stream(self._device)))

    def attend(self, batch: PagedBatch, q, scale: float | None = None, causal: bool = True, out=None, lse=None):
        """softmax(scale q K^T) V of a step's rows q [rows, heads, head dim] over their sequences' slots
        (scale 1 / sqrt(head dim) by default) and ln sum exp of the scores, float32 [rows, heads].
        Returns (out, lse), new tensors where they are not given; rows of no sequence are not written."""
        torch = _torch()
        if out is None:
            out = torch.empty_like(q)
        if lse is None:
            lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        a, b = _rows(q, "q", self._device), _rows(out, "out", self._device)
        at = _array(lse, "lse", "float32", self._device, q.shape[:2])
        ref = self._of(batch)
        space, size, _held = self._workspace(batch, "attention", a)
        check(library().jfh_paged_attention(self.ref, ref, ctypes.byref(a), a.head_dim ** -0.5 if scale is None else scale,
                                            int(causal), ctypes.byref(b), at, space, size, _stream(self._device)))
        return out, lse

    def weigh(self, batch: PagedBatch, q, lse, scale: float | None = None, causal: bool = True) -> None:
        """Adds the attention that the rows q (with attend's lse, scale and causal) give each position to
        the cache's weights."""
        a = _rows(q, "q", self._device)
        at = _array(lse, "lse", "float32", self._device, q.shape[:2])
        ref = self._of(batch)
        space, size, _held = self._workspace(batch, "weigh", a)
        check(library().jfh_paged_weigh(self.ref, ref, ctypes.byref(a), at, a.head_dim ** -0.5 if scale is None else scale,
                                        int(causal), space, size, _stream(self._device)))

    def evict(self, batch: PagedBatch, budget: int, n_first: int = 4, n_recent: int = 1) -> None:
        """Cuts every longer sequence to budget slots per K/V head: the positions below n_first, the
        n_recent newest, then the heaviest stay; batch.lengths becomes what is left."""
        budget = _count(budget, "budget")
        ref = self._of(batch)
        space, size, _held = self._workspace(batch, "evict", budget)
        check(library().jfh_paged_evict(self.ref, ref, budget, _count(n_first, "n_first"), _count(n_recent, "n_recent"), space,
                                        size, _stream(self._device)))
