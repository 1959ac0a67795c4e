"""Drafted tokens over a pool of 4-bit K/V pages: rotations, trees and their
verification, on torch CUDA tensors.

    rope = Rope(head_dim, base=500000.0)
    depth, mask = tree([-1, 0, 0, 1])                  # rows 1 and 2 hang on row 0, row 3 on row 1
    pool.extend([s], [4])
    q = pool.append_rope(layer, rope, q, k, v, [s], [4], depth=depth)
    o = pool.attend_tree(layer, q, [s], [4], mask)     # ... every layer
    kept, n_kept, nxt = verify(logits, tokens, parents, [4], u, u_next, temperature)
    pool.keep([s], [4], [kept[:n_kept[0]].tolist()])

Row 0 of a sequence's drafts is the token that was picked last, every other
row hangs on an earlier one.  Mirrors ecu_rope_* and ecu_draft_verify of
include/engine_cuda.h; the pool's part is in kv4.KvPool.  Work is enqueued on
`stream` (an int), by default torch's current stream of the tensors' device.
Errors raise EngineError.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from .engine import EngineError, int_list as _ints, last_error, lib
from .kv4 import _DTYPES, _at, _current, _total

ROWS = 64                      # drafted rows of a sequence, at most
_SCALING = {None: 0, "linear": 1, "bands": 2, "yarn": 3}


class EcuRope(C.Structure):
    _fields_ = [("rot", C.c_int), ("interleaved", C.c_int), ("factor", C.c_double), ("turn", C.c_uint64 * 64)]


class Rope:
    """A rotation of the first `rot` dimensions (by default all) of heads of head_dim (ecu_rope).

    base, and scaling "linear", "bands" or "yarn" by `factor` for contexts past `context` (slow, fast: turns over it;
    by default 1 and 4, of "yarn" 1 and 32); or freq, the radians a position of each pair, and then `factor`, which
    cosines and sines are multiplied by."""

    def __init__(self, head_dim: int, rot: int | None = None, interleaved: bool = False, base: float = 10000.0,
                 scaling: str | None = None, factor: float = 1.0, context: float = 0.0, slow: float = 1.0,
                 fast: float | None = None, freq=None):
        rot = head_dim if rot is None else rot
        _ints([head_dim, rot])
        if not 0 <= rot <= min(head_dim, 128):
            raise EngineError(f"{rot} turning dimensions of {head_dim}")
        self._r = EcuRope()
        self.at = C.addressof(self._r)
        if freq is not None:
            f = np.ascontiguousarray(freq, dtype=np.float64)
            if scaling is not None or f.ndim != 1 or len(f) != rot // 2:
                raise EngineError(f"freq: {rot // 2} frequencies without a scaling are wanted")
            rc = lib().ecu_rope_set(self.at, rot, int(interleaved), f.ctypes.data, float(factor))
        else:
            if scaling not in _SCALING:
                raise EngineError(f"no scaling {scaling!r}")
            fast = (32.0 if scaling == "yarn" else 4.0) if fast is None else fast
            rc = lib().ecu_rope_init(self.at, rot, int(interleaved), float(base), _SCALING[scaling], float(factor),
                                     float(context), float(slow), float(fast))
        if rc != 0:
            raise EngineError(last_error())

    @property
    def rot(self) -> int:
        return int(self._r.rot)

    @property
    def factor(self) -> float:
        """What cosines and sines are multiplied by."""
        return float(self._r.factor)

    @property
    def turns(self) -> np.ndarray:
        """Turns a position of each pair, in units of 2^-64 (uint64)."""
        return np.array(self._r.turn[:self.rot // 2], dtype=np.uint64)


def tree(parents, device: int | None = 0):
    """(depth, mask) of drafted rows, for append_rope and attend_tree: parents is one list, or a list of lists (one a
    sequence), of each row's parent, -1 for none.  int32 and int64 tensors on the device (None: numpy arrays)."""
    try:
        lists = [parents] if len(parents) and np.ndim(parents[0]) == 0 else parents
        lists = [(p, len(p)) for p in lists]
    except TypeError:
        raise EngineError("parents: a list of whole numbers, or a list of such lists, is wanted") from None
    depth, mask = [], []
    for p, n in lists:
        p = _ints(p) if n else np.zeros(0, np.int32)
        if n > ROWS:
            raise EngineError(f"{n} drafted rows of a sequence ({ROWS} at most)")
        d, m = [], []
        for j, up in enumerate(p.tolist()):
            if not -1 <= up < j:
                raise EngineError(f"row {j} cannot hang on row {up}")
            d.append(d[up] + 1 if up >= 0 else 0)
            m.append((m[up] if up >= 0 else 0) | 1 << j)
        depth += d
        mask += m
    depth = np.array(depth, dtype=np.int32)
    mask = np.array(mask, dtype=np.uint64).view(np.int64)
    if device is None:
        return depth, mask
    return torch.from_numpy(depth).to(f"cuda:{device}"), torch.from_numpy(mask).to(f"cuda:{device}")


def _vector(t: torch.Tensor | None, what: str, dtype: torch.dtype, n: int, dev: int) -> int | None:
    if t is None:
        return None
    if t.dtype is not dtype or t.dim() != 1 or t.numel() != n or not t.is_contiguous() or t.get_device() != dev:
        raise EngineError(f"{what}: {n} contiguous {str(dtype)[6:]} numbers on CUDA device {dev} are wanted")
    return t.data_ptr()


def _matrix(t: torch.Tensor, what: str, rows: int) -> int:
    """The row stride of [rows, n_vocab]."""
    if not t.is_cuda or t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise EngineError(f"{what}: {rows} rows of a vocabulary on a CUDA device are wanted")
    return t.stride(0) if rows > 1 else t.shape[1]


def verify(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, n_row, u: torch.Tensor, u_next: torch.Tensor,
           temperature: torch.Tensor | None = None, draft: torch.Tensor | None = None, kept: torch.Tensor | None = None,
           n_kept: torch.Tensor | None = None, next: torch.Tensor | None = None, stream: int | None = None):
    """(kept, n_kept, next) of drafted tokens (ecu_draft_verify): logits [rows, n_vocab] of all sequences' rows, n_row[i]
    (host) of them the i-th sequence's; tokens, parents (int32) and u (float32), one a row; u_next and temperature
    (float32; 0: greedy), one a sequence; draft [rows, n_vocab] (float32), the distributions that a row's children were
    drawn from.  kept (one a row), n_kept and next (one a sequence) are int32."""
    cnt = _ints(n_row)
    n, rows = len(cnt), _total(cnt)
    ls = _matrix(logits, "logits", rows)
    dev, vocab = logits.get_device(), logits.shape[1]
    if logits.dtype not in _DTYPES:
        raise EngineError("logits: float32, float16 or bfloat16 is wanted")
    ds, dp = 0, None
    if draft is not None:
        ds, dp = _matrix(draft, "draft", rows), draft.data_ptr()
        if draft.dtype != torch.float32 or draft.shape[1] != vocab or draft.get_device() != dev:
            raise EngineError("draft: float32 rows of the logits' vocabulary and device are wanted")
    if u is None or u_next is None or tokens is None or parents is None:
        raise EngineError("tokens, parents, u and u_next are wanted")
    where = f"cuda:{dev}"
    kept = torch.empty(rows, dtype=torch.int32, device=where) if kept is None else kept
    n_kept = torch.empty(n, dtype=torch.int32, device=where) if n_kept is None else n_kept
    next = torch.empty(n, dtype=torch.int32, device=where) if next is None else next
    i32, f32 = torch.int32, torch.float32
    if lib().ecu_draft_verify(_DTYPES[logits.dtype], logits.data_ptr(), ls, vocab, dp, ds, _vector(tokens, "tokens", i32, rows, dev),
                              _vector(parents, "parents", i32, rows, dev), _at(cnt), n, _vector(u, "u", f32, rows, dev),
                              _vector(u_next, "u_next", f32, n, dev), _vector(temperature, "temperature", f32, n, dev),
                              _vector(kept, "kept", i32, rows, dev), _vector(n_kept, "n_kept", i32, n, dev),
                              _vector(next, "next", i32, n, dev), dev, _current(dev) if stream is None else stream) != 0:
        raise EngineError(last_error())
    return kept, n_kept, next
