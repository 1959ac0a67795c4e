"""A pool of 4-bit K/V pages shared by many sequences, and the attention over
it and over packed prompts, on torch CUDA tensors.

    pool = KvPool(n_layer, n_head_kv, head_dim, n_pages, n_seq, max_pages)
    pool.extend([0], [n])                      # n new positions of sequence 0
    pool.append(layer, k, v, [0], [n])         # their K and V rows
    prompt_attention(q, k, v, [0, n])          # the prompt over itself
    pool.fork([0], [1])                        # sequence 1 shares its pages
    pool.attend(layer, q, [0, 1])              # one query row a sequence

The classes mirror ecu_kv_* and ecu_attn_prompt of include/engine_cuda.h name
for name (the layout of a page is described there).  Rows are tensors
[rows, heads, head_dim] (or [rows, heads * head_dim]) whose heads lie one
after the other, the rows any distance apart.  Lists of sequences and counts
are host lists or numpy arrays.  Work is enqueued on `stream` (an int), by
default torch's current stream of the tensors' device.  Errors raise
EngineError.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from .engine import EcuKvInfo, EngineError, int_list as _ints, last_error, lib

PAGE = 64
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def page_bytes(n_head_kv: int, head_dim: int) -> int:
    """Bytes of one page of one layer (0: a shape that is not covered)."""
    _ints([n_head_kv, head_dim])
    return int(lib().ecu_kv4_page_bytes(n_head_kv, head_dim))


_INT_AT = C.c_int.from_buffer


def _at(a: np.ndarray) -> int:
    """The address of an array's numbers."""
    try:
        return C.addressof(_INT_AT(a))        # a third of what a.ctypes.data takes
    except (TypeError, ValueError):           # read-only, or empty
        return a.ctypes.data


def _row(t: torch.Tensor, what: str, heads: int | None, hd: int, device: int) -> tuple[int, int]:
    """(heads, row stride) of rows [n, heads, hd] or [n, heads * hd]."""
    if t.dtype not in _DTYPES or not t.is_cuda or t.get_device() != device:
        raise EngineError(f"{what}: rows of float32, float16 or bfloat16 on CUDA device {device} are wanted")
    shape, st = t.shape, t.stride()
    if len(shape) == 3:
        h = shape[1]
        good = shape[2] == hd and st[2] == 1 and (st[1] == hd or h == 1)
    else:
        good = len(shape) == 2 and shape[1] % hd == 0 and st[1] == 1
        h = shape[1] // hd if good else 0
    if not good or h < 1 or (heads is not None and h != heads):
        raise EngineError(f"{what}: rows {tuple(shape)} with strides {st} are not [n, "
                          f"{'heads' if heads is None else heads}, {hd}] with their heads one after the other")
    return h, st[0] if shape[0] > 1 else h * hd


def _current(device: int) -> int:
    """torch's current stream of a device."""
    return torch._C._cuda_getCurrentRawStream(device)


def _like(t: torch.Tensor, of: torch.Tensor) -> bool:
    """Of the type, device, shape and strides of another, which has been checked."""
    return t.dtype is of.dtype and t.shape == of.shape and t.stride() == of.stride() and t.is_cuda and \
        t.get_device() == of.get_device()


class _Memory:
    """Device memory as torch.as_tensor takes it."""

    def __init__(self, ptr: int, shape: tuple, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<i4", "data": (ptr, False), "version": 3,
                                         "strides": None, "stream": None}


class KvPool:
    """A pool of 4-bit K/V pages (ecu_kv)."""

    def __init__(self, n_layer: int, n_head_kv: int, head_dim: int, n_pages: int, n_seq: int, max_pages: int,
                 device: int = 0, data: torch.Tensor | None = None):
        """data: the pages' memory (n_layer * n_pages * page_bytes(), kept by
        the pool as long as it lives), else the pool allocates it.  device -1:
        the bookkeeping alone."""
        self.h = C.c_void_p()
        _ints([n_layer, n_head_kv, head_dim, n_pages, n_seq, max_pages, device])      # (ctypes drops higher bits)
        if data is not None:
            want = n_layer * n_pages * page_bytes(n_head_kv, head_dim)
            if device < 0 or not data.is_cuda or data.get_device() != device or not data.is_contiguous() or \
                    data.numel() * data.element_size() < want:
                raise EngineError(f"data: {want} contiguous bytes on CUDA device {device} are wanted")
        err = C.create_string_buffer(512)
        rc = lib().ecu_kv_open(C.byref(self.h), n_layer, n_head_kv, head_dim, n_pages, n_seq, max_pages, device,
                               data.data_ptr() if data is not None else None, err, 512)
        if rc != 0:
            raise EngineError(err.value.decode(errors="replace") or last_error())
        self.data = data
        i = self.info()
        self.n_layer, self.n_head_kv, self.head_dim = i.n_layer, i.n_head_kv, i.head_dim
        self.n_pages, self.n_seq, self.max_pages, self.device = i.n_pages, i.n_seq, i.max_pages, i.device
        self._table, self._len = i.table, i.len

    def info(self) -> EcuKvInfo:
        i = EcuKvInfo()
        if lib().ecu_kv_get_info(self.h, C.byref(i)) != 0:
            raise EngineError("the pool is closed")
        return i

    @property
    def used(self) -> int:
        """Pages that some sequence holds."""
        return int(self.info().used)

    @property
    def table(self) -> torch.Tensor:
        """The device's page ids [n_seq, max_pages], -1 where there is none (a view: for reading)."""
        self.info()
        return torch.as_tensor(_Memory(self._table, (self.n_seq, self.max_pages), self), device=f"cuda:{self.device}")

    @property
    def lengths(self) -> torch.Tensor:
        """The device's positions of each sequence [n_seq] (a view: for reading)."""
        self.info()
        return torch.as_tensor(_Memory(self._len, (self.n_seq,), self), device=f"cuda:{self.device}")

    def length(self, seq: int) -> int:
        _ints([seq])
        n = int(lib().ecu_kv_len(self.h, int(seq), None, 0))
        if n < 0:
            raise EngineError(last_error())
        return n

    def pages(self, seq: int) -> list[int]:
        buf = np.zeros((self.length(seq) + PAGE - 1) // PAGE, dtype=np.int32)
        lib().ecu_kv_len(self.h, int(seq), buf.ctypes.data, len(buf))
        return [int(p) for p in buf]

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.n_layer:
            raise EngineError(f"layer {layer} of {self.n_layer}")
        return layer

    def _stream(self, stream):
        if stream is not None or self.device < 0:
            return stream
        return _current(self.device)

    def _change(self, f, a, b, stream) -> None:
        a, b = _ints(a), _ints(b)
        if len(a) != len(b):
            raise EngineError(f"{len(a)} sequences and {len(b)} values for them")
        if f(self.h, _at(a), _at(b), len(a), self._stream(stream)) != 0:
            raise EngineError(last_error())

    def extend(self, seq, n_new, stream: int | None = None) -> None:
        """Sequences grow by n_new positions (pages taken; a shared, partly filled last page copied)."""
        self._change(lib().ecu_kv_extend, seq, n_new, stream)

    def fork(self, src, dst, stream: int | None = None) -> None:
        """Empty slots dst become copies of src that share its pages."""
        self._change(lib().ecu_kv_fork, src, dst, stream)

    def truncate(self, seq, length, stream: int | None = None) -> None:
        """Sequences keep their first `length` positions."""
        self._change(lib().ecu_kv_truncate, seq, length, stream)

    def free(self, seq, stream: int | None = None) -> None:
        a = _ints(seq)
        if lib().ecu_kv_free(self.h, _at(a), len(a), self._stream(stream)) != 0:
            raise EngineError(last_error())

    def compact(self, stream: int | None = None) -> int:
        """Pages in use move to ids 0..used-1; the number moved."""
        n = int(lib().ecu_kv_compact(self.h, self._stream(stream)))
        if n < 0:
            raise EngineError(last_error())
        return n

    def inject_failure(self, launch: int = 0) -> None:
        """The launch-th device update of the next change fails (ecu_kv_inject_failure): failure-path testing."""
        _ints([launch])
        if lib().ecu_kv_inject_failure(self.h, launch) != 0:
            raise EngineError(last_error())

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, seq, n_new, k_out: torch.Tensor | None = None,
               v_out: torch.Tensor | None = None, stream: int | None = None) -> None:
        """The newest n_new[i] positions' rows of sequences seq[i] (ecu_kv_append); k_out, v_out: contiguous
        rows that receive the values as the cache holds them."""
        heads, hd, dev = self.n_head_kv, self.head_dim, self.device
        _, ks = _row(k, "k", heads, hd, dev)
        vs = ks if _like(v, k) else _row(v, "v", heads, hd, dev)[1]
        n_new = _ints(n_new)
        s = None if seq is None else _ints(seq)
        n = len(n_new)
        rows = sum(n_new.tolist()) if n <= 256 else int(n_new.sum(dtype=np.int64))
        if (s is not None and len(s) != n) or k.shape[0] != rows or v.shape[0] != rows or k.dtype != v.dtype:
            raise EngineError(f"k and v: {rows} rows of one type are wanted, and a count for each sequence")
        if (k_out is None) != (v_out is None):
            raise EngineError("k_out and v_out come together")
        ko = vo = None
        od = k.dtype
        if k_out is not None:
            _row(k_out, "k_out", heads, hd, dev)
            if not _like(v_out, k_out):
                _row(v_out, "v_out", heads, hd, dev)
            if k_out.shape[0] != rows or v_out.shape[0] != rows or k_out.dtype != v_out.dtype or \
                    not k_out.is_contiguous() or not v_out.is_contiguous():
                raise EngineError(f"k_out and v_out: {rows} contiguous rows of one type are wanted")
            ko, vo, od = k_out.data_ptr(), v_out.data_ptr(), k_out.dtype
        if lib().ecu_kv_append(self.h, self._layer(layer), _DTYPES[k.dtype], k.data_ptr(), v.data_ptr(), ks, vs,
                               None if s is None else _at(s), _at(n_new), n, _DTYPES[od], ko, vo,
                               self._stream(stream)) != 0:
            raise EngineError(last_error())

    def attend(self, layer: int, q: torch.Tensor, seq=None, out: torch.Tensor | None = None, scale: float | None = None,
               ws: torch.Tensor | None = None, stream: int | None = None) -> torch.Tensor:
        """One query row per sequence over all of its positions (ecu_kv_attend); ws: workspace() for calls that
        are captured or may overlap."""
        heads, qs = _row(q, "q", None, self.head_dim, self.device)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        os_ = qs if _like(out, q) else _row(out, "out", heads, self.head_dim, self.device)[1]
        s = None if seq is None else _ints(seq)
        if out.dtype != q.dtype or out.shape[0] != q.shape[0] or (s is not None and len(s) != q.shape[0]):
            raise EngineError("out and the sequences: one for each row of q, of its type")
        if ws is not None and (not ws.is_cuda or ws.get_device() != self.device or not ws.is_contiguous() or
                               ws.numel() * ws.element_size() < self.ws_bytes()):
            raise EngineError(f"ws: {self.ws_bytes()} contiguous bytes on CUDA device {self.device} are wanted")
        if lib().ecu_kv_attend(self.h, self._layer(layer), _DTYPES[q.dtype], q.data_ptr(), out.data_ptr(), heads, qs, os_,
                               None if s is None else _at(s), q.shape[0],
                               self.head_dim ** -0.5 if scale is None else scale,
                               None if ws is None else ws.data_ptr(), self._stream(stream)) != 0:
            raise EngineError(last_error())
        return out

    def ws_bytes(self) -> int:
        return int(lib().ecu_kv_ws_bytes(self.h))

    def workspace(self) -> torch.Tensor:
        """A workspace for attend."""
        return torch.zeros(self.ws_bytes(), dtype=torch.uint8, device=f"cuda:{self.device}")

    def read(self, layer: int, seq: int, pos: int = 0, n: int | None = None, stream: int | None = None):
        """(K, V) rows [n, n_head_kv, head_dim] of cached positions as numpy arrays (ecu_kv_read)."""
        n = self.length(seq) - pos if n is None else n
        _ints([pos, n])
        k, v = (np.empty((max(n, 0), self.n_head_kv, self.head_dim), dtype=np.float32) for _ in range(2))
        if lib().ecu_kv_read(self.h, self._layer(layer), int(seq), pos, n, k.ctypes.data, v.ctypes.data, self._stream(stream)) != 0:
            raise EngineError(last_error())
        return k, v

    def close(self) -> None:
        if self.h:
            lib().ecu_kv_close(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q, cu_k=None, out: torch.Tensor | None = None,
                     scale: float | None = None, stream: int | None = None) -> torch.Tensor:
    """Causal attention of packed prompts (ecu_attn_prompt): q [rows, n_head, head_dim], k and v [rows, n_head_kv,
    head_dim], offsets cu_q (and cu_k, where sequences have more keys than queries) of each sequence's rows."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3 or not q.is_cuda:
        raise EngineError("q, k and v: CUDA tensors [rows, heads, head_dim] are wanted")
    dev, hd = q.get_device(), q.shape[2]
    heads, qs = _row(q, "q", None, hd, dev)
    kv, ks = _row(k, "k", None, hd, dev)
    vs = ks if _like(v, k) else _row(v, "v", kv, hd, dev)[1]
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    os_ = qs if _like(out, q) else _row(out, "out", heads, hd, dev)[1]
    cq = _ints(cu_q)
    ck = cq if cu_k is None else _ints(cu_k)
    if q.dtype != k.dtype or q.dtype != v.dtype or q.dtype != out.dtype or out.shape[0] != q.shape[0]:
        raise EngineError("q, k, v and out of one type, out with q's rows, are wanted")
    if len(cq) < 1 or len(cq) != len(ck) or cq[-1] != q.shape[0] or ck[-1] != k.shape[0] or k.shape[0] != v.shape[0]:
        raise EngineError("cu_q and cu_k: one offset more than sequences, the last one the rows of q and of k and v")
    if stream is None:
        stream = _current(dev)
    if lib().ecu_attn_prompt(_DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), heads, kv, hd, qs,
                             ks, vs, os_, _at(cq), _at(ck), len(cq) - 1,
                             hd ** -0.5 if scale is None else scale, dev, stream) != 0:
        raise EngineError(last_error())
    return out


def prompt_status(device: int = 0, stream: int | None = None) -> None:
    """Waits for the stream's work; raises where a prompt attention on the device gave up on a wait since this was
    last asked: its rows are NaN (ecu_attn_prompt_status)."""
    if lib().ecu_attn_prompt_status(device, _current(device) if stream is None else stream) != 0:
        raise EngineError(last_error())
