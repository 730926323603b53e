"""Operators of the towers and encoders beside the text model, on device buffers
(the operator part of include/svl_gpu.h).

* ``AxisRope``       -- rotary positions with up to four axes (time, height,
                        width ...) over query and key rows.
* ``AttentionPlan``  -- attention over packed sequences with capped scores, a
                        distance bias, document, prefix, order and window masks.
* ``Q4Weight``       -- a weight matrix in 4 bits and its product with a few rows.

They make the soft tokens that ``TextModel.forward_with_features`` takes, or
another encoder's rows: project, rotate, attend, project.  Device buffers are
passed as addresses (``tensor.data_ptr()``) with row strides in elements; calls
queue on ``stream`` (a ``cudaStream_t`` as an int, 0 = the legacy default
stream) and return.  A handle belongs to its device, may be shared by threads,
streams and captured graphs, and has to outlive the work that was queued with
it.  ``close()``, and the last reference to a handle that was not closed, frees
its device memory: that may wait for the device, and may happen while a graph
is being captured.  Creating a handle may not.
"""

from __future__ import annotations

import ctypes
import threading

import numpy as np

from . import errors
from ._abi import (
    DTYPE_BF16,
    DTYPE_F16,
    DTYPE_F32,
    ErrBuf,
    SvlAttentionConfig,
    SvlRopeConfig,
    load_library,
    tensor_views,
)

_P = ctypes.c_void_p

DTYPES = {"f32": DTYPE_F32, "bf16": DTYPE_BF16, "f16": DTYPE_F16}
ARRANGEMENTS = {"split": 0, "sections": 1, "interleaved": 2}


def _dtype(name: str) -> int:
    if name not in DTYPES:
        raise errors.UsageError(f"unknown dtype {name!r} (f32, bf16 or f16)")
    return DTYPES[name]


def _count(value, what: str, most: int = (1 << 32) - 1) -> int:
    """A whole number that fits its C argument (ctypes would cut it)."""
    try:
        n = int(value)
    except (ValueError, OverflowError):  # NaN, infinities
        n = -1
    if n != value or not 0 <= n <= most:
        raise errors.UsageError(f"{what} must be a whole number in 0..={most}")
    return n


def _whole(values, dtype, what: str) -> np.ndarray:
    """A flat array of whole numbers in ``dtype``, refused where one does not fit."""
    a = np.asarray(values)
    if a.size and a.dtype.kind not in "iu":
        raise errors.UsageError(f"{what} must be whole numbers")
    info = np.iinfo(dtype)
    if a.size and (int(a.min()) < info.min or int(a.max()) > info.max):
        raise errors.UsageError(f"{what} are outside {info.min}..={info.max}")
    return np.ascontiguousarray(a.ravel(), dtype)


def _ptr(a):
    return None if a is None else a.ctypes.data


class _PerThread(threading.local):
    """One message buffer a thread for the calls on device buffers, which are short."""

    def __init__(self):
        self.err = ErrBuf()


_thread = _PerThread()


class _Handle:
    _h = None
    _destroy = ""

    def close(self):
        if getattr(self, "_h", None):
            getattr(self._lib, self._destroy)(self._h)
            self._h = None

    def __del__(self):
        self.close()

    @property
    def handle(self):
        return self._h


class AxisRope(_Handle):
    """``pairs[a]`` pairs of a head's dimensions turn with axis ``a``.

    arrangement "split": each axis owns its own ``2 * pairs[a]`` dimensions,
    rotate-half inside them, base ``theta[a]``.  "sections" / "interleaved": one
    rotate-half over all pairs with base ``theta[0]``; the axes own runs of
    pairs, or take them in turn.  Dimensions behind the pairs are copied.  Bases
    are at least 1/128."""

    _destroy = "svl_rope_destroy"

    def __init__(self, head_dim: int, pairs, theta=10000.0, arrangement: str = "split"):
        if arrangement not in ARRANGEMENTS:
            raise errors.UsageError(f"unknown arrangement {arrangement!r} (split, sections or interleaved)")
        pairs = [_count(p, "pairs") for p in pairs]
        thetas = [float(theta)] * len(pairs) if np.ndim(theta) == 0 else [float(t) for t in theta]
        if not 1 <= len(pairs) <= 4:
            raise errors.UsageError("n_axes is outside 1..=4")
        if len(thetas) not in (1, len(pairs)) or (len(thetas) == 1 and arrangement == "split" and len(pairs) > 1):
            raise errors.UsageError("theta needs one value, or one for each axis")
        self._lib = load_library()
        c = SvlRopeConfig(head_dim=_count(head_dim, "head_dim"), n_axes=len(pairs),
                          arrangement=ARRANGEMENTS[arrangement])
        c.pairs[: len(pairs)] = pairs
        c.theta[: len(thetas)] = thetas
        h, eb = _P(), ErrBuf()
        eb.check(self._lib.svl_rope_create(ctypes.byref(c), ctypes.byref(h), *eb.args))
        self._h = h
        self.head_dim = head_dim
        self.n_axes = len(pairs)

    def apply_device(self, dtype: str, positions: int, n_tokens: int, q: int, ld_q: int, q_heads: int, q_out: int,
                     ld_q_out: int, k: int = 0, ld_k: int = 0, k_heads: int = 0, k_out: int = 0, ld_k_out: int = 0,
                     device: int = 0, stream: int = 0) -> None:
        """Rotates ``n_tokens`` rows of ``q_heads`` and ``k_heads`` heads; ``positions``
        holds ``n_axes`` x ``n_tokens`` int32.  In place where an output is its input."""
        if (q_heads | k_heads) >> 32:  # ctypes would cut them
            raise errors.UsageError("more than 65535 heads")
        eb = _thread.err
        rc = self._lib.svl_rope_apply_device(self._h, device, _dtype(dtype), positions, n_tokens, q, ld_q, q_heads,
                                             q_out, ld_q_out, k, ld_k, k_heads, k_out, ld_k_out, stream or None,
                                             *eb.args)
        if rc:
            eb.check(rc)


class AttentionPlan(_Handle):
    """The layout and masks of a packed batch (``svl_attention_plan_create``),
    shared by every layer that attends over it.

    ``cu_q`` / ``cu_k``: offsets (batch + 1; ``cu_k`` None = ``cu_q``).  Query i of a
    sequence sits at position i + n_k - n_q.  ``cap`` > 0 caps scores by
    cap * tanh(score / cap); ``slopes`` (one a query head) subtract
    slope * |distance|; ``prefix``: keys of each sequence that all its rows see;
    ``doc_q`` / ``doc_k``: the document of every row, negative = padding;
    ``window``: the largest visible distance.  A row that sees no key is zero
    with a log sum of -inf."""

    _destroy = "svl_attention_plan_destroy"

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, cu_q, cu_k=None, *, dtype: str = "bf16",
                 scale: float | None = None, cap: float = 0.0, causal: bool = False, window: int | None = None,
                 prefix=None, doc_q=None, doc_k=None, slopes=None, device: int = 0):
        if window is not None:
            window = _count(window, "window", (1 << 31) - 1)
        head_dim = _count(head_dim, "head_dim")
        if cap and not ctypes.c_float(cap).value:
            raise errors.UsageError("cap is neither 0 nor in 1e-30..=1e30")
        c = SvlAttentionConfig(dtype=_dtype(dtype), q_heads=_count(q_heads, "q_heads"),
                               kv_heads=_count(kv_heads, "kv_heads"), head_dim=head_dim,
                               scale=float(max(head_dim, 1) ** -0.5 if scale is None else scale), cap=float(cap),
                               causal=int(bool(causal)), window=-1 if window is None else window)
        cq = _whole(cu_q, np.uint64, "cu_q")
        ck = None if cu_k is None else _whole(cu_k, np.uint64, "cu_k")
        if not cq.size or (ck is not None and ck.size != cq.size):
            raise errors.UsageError("offsets must hold batch + 1 entries")
        n_q, n_k = int(cq[-1]), int((cq if ck is None else ck)[-1])
        pre = None if prefix is None else _whole(prefix, np.uint64, "prefix")
        dq = None if doc_q is None else _whole(doc_q, np.int32, "doc_q")
        dk = None if doc_k is None else _whole(doc_k, np.int32, "doc_k")
        sl = None if slopes is None else np.ascontiguousarray(np.asarray(slopes, np.float32).ravel())
        for a, n, what in ((pre, cq.size - 1, "prefix"), (dq, n_q, "doc_q"), (dk, n_k, "doc_k"),
                           (sl, q_heads, "slopes")):
            if a is not None and a.size != n:
                raise errors.UsageError(f"{what} must hold {n} entries")
        self._lib = load_library()
        h, eb = _P(), ErrBuf()
        eb.check(self._lib.svl_attention_plan_create(device, ctypes.byref(c), _ptr(cq), _ptr(ck), cq.size - 1,
                                                     _ptr(pre), _ptr(dq), _ptr(dk), _ptr(sl), ctypes.byref(h),
                                                     *eb.args))
        self._h = h
        self.device = device
        n = ctypes.c_uint64()
        self._lib.svl_attention_plan_workspace(h, ctypes.byref(n))
        #: bytes that run_device needs as its workspace (may be 0)
        self.workspace_bytes = n.value

    def run_device(self, q: int, ld_q: int, k: int, ld_k: int, v: int, ld_v: int, out: int, ld_out: int, lse: int = 0,
                   workspace: int = 0, workspace_bytes: int = 0, stream: int = 0) -> None:
        """One attention over the batch; ``lse`` (optional): q rows x q_heads float32."""
        eb = _thread.err
        rc = self._lib.svl_attention_device(self._h, q, ld_q, k, ld_k, v, ld_v, out, ld_out, lse or None,
                                            workspace or None, workspace_bytes, stream or None, *eb.args)
        if rc:
            eb.check(rc)

    def check(self) -> None:
        """Synchronises and reports a deferred device-side error."""
        eb = ErrBuf()
        eb.check(self._lib.svl_attention_check(self._h, *eb.args))


class Q4Weight(_Handle):
    """A weight matrix [n, k] in 4 bits, (code - zero) * scale per group of columns."""

    _destroy = "svl_q4_destroy"

    def __init__(self, handle, device: int):
        self._lib = load_library()
        self._h = handle
        self.device = device
        n, k, group, kind = (ctypes.c_uint32() for _ in range(4))
        eb = ErrBuf()
        eb.check(self._lib.svl_q4_read(handle, ctypes.byref(n), ctypes.byref(k), ctypes.byref(group),
                                       ctypes.byref(kind), None, None, None, *eb.args))
        self.n, self.k, self.group = n.value, k.value, group.value
        self.scale_dtype = "f16" if kind.value == DTYPE_F16 else "bf16"

    @classmethod
    def from_codes(cls, codes: int, scales: int, n: int, k: int, group: int, zeros: int = 0,
                   scale_dtype: str = "bf16", device: int = 0) -> "Q4Weight":
        """From codes [n, k/2] (column 2c in the low half of byte c), scales and zeros
        [n, k/group], given as addresses of host or device memory."""
        lib, h, eb = load_library(), _P(), ErrBuf()
        eb.check(lib.svl_q4_create(device, codes, scales, _dtype(scale_dtype), zeros or None, _count(n, "n"),
                                   _count(k, "k"), _count(group, "group"), ctypes.byref(h), *eb.args))
        return cls(h, device)

    @classmethod
    def quantize(cls, weight, group: int = 64, asymmetric: bool = False, device: int = 0) -> "Q4Weight":
        """Quantises a host weight (an array, or a Safetensors entry in F32 or BF16)."""
        views, keep = tensor_views({"weight": weight})
        lib, h, eb = load_library(), _P(), ErrBuf()
        eb.check(lib.svl_q4_quantize(device, views, _count(group, "group"), int(bool(asymmetric)), ctypes.byref(h),
                                     *eb.args))
        del keep
        return cls(h, device)

    def read(self):
        """(codes uint8 [n, k/2], scales uint16 bits [n, k/group], zeros uint8 [n, k/group])."""
        codes = np.empty((self.n, self.k // 2), np.uint8)
        scales = np.empty((self.n, self.k // self.group), np.uint16)
        zeros = np.empty_like(scales, dtype=np.uint8)
        eb = ErrBuf()
        eb.check(self._lib.svl_q4_read(self._h, None, None, None, None, _ptr(codes), _ptr(scales), _ptr(zeros),
                                       *eb.args))
        return codes, scales, zeros

    def linear_device(self, dtype: str, x: int, ld_x: int, rows: int, y: int, ld_y: int, stream: int = 0) -> None:
        """y = x W^T for ``rows`` rows."""
        eb = _thread.err
        rc = self._lib.svl_q4_linear_device(self._h, _dtype(dtype), x, ld_x, rows, y, ld_y, stream or None, *eb.args)
        if rc:
            eb.check(rc)
