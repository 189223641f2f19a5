"""LogitOps: operators over rows of class logits (include/tmnn_hip.h, class
logits): log-probabilities of given classes with rank, entropy and the best
alternatives, their gradient, and distillation from a teacher's top values.

Arrays are numpy arrays (copied in and out; the results are there on return) or
device tensors (anything with data_ptr(), shape, stride() and dtype, as torch's;
the call is only enqueued, on the tensors' current torch stream unless `stream`
says otherwise). All arrays of a call are of one sort. Logits are float32,
float16 or (device) bfloat16, [rows, classes] with unit stride within a row;
class ids int32 or int64; everything else float32 / int32 and contiguous.
No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import struct
import sys

import numpy as np

from . import _lib
from .trainer import ClosedError, DTypeError, _Context

_PACK_LOGPROBS = struct.Struct("=Iiii4q12Qfi")
_PACK_DISTILL = struct.Struct("=Iiii4q7Qif")
_SIZE_LOGPROBS, _SIZE_DISTILL = _PACK_LOGPROBS.size, _PACK_DISTILL.size
_DTYPE_NAMES: dict = {}  # dtype object -> its name


def _name(dtype) -> str:
    """'float32' of numpy's and torch's float32 alike."""
    got = _DTYPE_NAMES.get(dtype)
    if got is None:
        got = _DTYPE_NAMES[dtype] = str(dtype).replace("torch.", "")
    return got


def _on_device(x) -> bool:
    return hasattr(x, "data_ptr")


class _Call:
    """The arrays of one call: all on the host or all on one device."""

    __slots__ = ("device", "ordinal", "shape", "dtype", "stride")

    def __init__(self, logits, name: str, ordinal: int):
        self.device = _on_device(logits)
        self.ordinal = ordinal
        if not self.device and not isinstance(logits, np.ndarray):
            raise TypeError(f"{name} must be a numpy array or a device tensor")
        dtype = _name(logits.dtype)
        if dtype not in _lib.DTYPES:
            raise DTypeError(f"{name} must be float32, float16 or bfloat16, got {dtype}")
        self.dtype = dtype
        self.shape = shape = tuple(logits.shape)
        if len(shape) != 2:
            raise ValueError(f"{name} must be 2D (rows, classes)")
        if shape[1] < 1:
            raise ValueError(f"{name} must have at least one class")
        self.stride = self._row_stride(logits, name)

    def _row_stride(self, x, name: str) -> int:
        rows, classes = self.shape
        if self.device:
            self._check_place(x, name)
            row, col = x.stride()
        else:
            size = x.itemsize
            row, col = (s // size if s % size == 0 else -1 for s in x.strides)
        if rows == 0:
            return classes
        if col != 1 and classes > 1:
            raise ValueError(f"{name} must have unit stride within a row")
        if rows == 1:
            return max(row, classes)
        if row < classes:
            raise ValueError(f"{name} must have rows that do not overlap")
        return row

    def _check_place(self, x, name: str) -> None:
        d = x.device
        if d.type != "cuda" or (d.index or 0) != self.ordinal:
            raise ValueError(f"{name} must be on device {self.ordinal}, is on {d}")

    def address(self, x) -> int:
        return x.data_ptr() if self.device else x.ctypes.data

    def array(self, x, name: str, shape: tuple, dtypes) -> int:
        """The address of a contiguous array of this shape and one of these types."""
        if _on_device(x) != self.device or not (self.device or isinstance(x, np.ndarray)):
            raise TypeError(f"{name} must be {'a device tensor' if self.device else 'a numpy array'}"
                            ", as the logits are")
        if _name(x.dtype) not in dtypes:
            raise DTypeError(f"{name} must be {' or '.join(dtypes)}, got {_name(x.dtype)}")
        if tuple(x.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")
        if self.device:
            if x.device.type != "cuda" or (x.device.index or 0) != self.ordinal:
                self._check_place(x, name)
            if not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            return x.data_ptr()
        if not x.flags["C_CONTIGUOUS"]:
            raise ValueError(f"{name} must be contiguous")
        return x.ctypes.data

    def matrix(self, x, name: str) -> tuple[int, int]:
        """Address and row stride of a second matrix like the logits."""
        if _on_device(x) != self.device or not (self.device or isinstance(x, np.ndarray)):
            raise TypeError(f"{name} must be {'a device tensor' if self.device else 'a numpy array'}"
                            ", as the logits are")
        if _name(x.dtype) != self.dtype:
            raise DTypeError(f"{name} must be {self.dtype} as the logits, got {_name(x.dtype)}")
        if tuple(x.shape) != self.shape:
            raise ValueError(f"{name} must have shape {self.shape}, got {tuple(x.shape)}")
        return self.address(x), self._row_stride(x, name)

    def empty(self, shape: tuple, dtype: str):
        if not self.device:
            return np.empty(shape, dtype)
        torch = sys.modules["torch"]
        return torch.empty(shape, dtype=getattr(torch, dtype), device=f"cuda:{self.ordinal}")

    def output(self, out: dict, key: str, shape: tuple, dtype: str, align: int = 1) -> int:
        x = out.get(key)
        if x is None:
            x = out[key] = self.empty(shape, dtype)
        at = self.array(x, f"out[{key!r}]", shape, (dtype,))
        if at % align:
            raise ValueError(f"out[{key!r}] must be {align}-byte aligned")
        return at

    def d_logits(self, out) -> tuple:
        if out is None:
            out = self.empty(self.shape, self.dtype)
        return (out, *self.matrix(out, "d_logits"))


_F32, _I32, _IDS = ("float32",), ("int32",), ("int32", "int64")


def _optional(call: _Call, x, name: str, shape: tuple, dtypes=_F32) -> int:
    return 0 if x is None else call.array(x, name, shape, dtypes)


class LogitOps:
    """Operators over rows of class logits on one device.

    Holds the workspace of its calls: calls through one object are ordered where
    they share it, also across streams. Use one object per thread, and one of its
    own for a stream that is captured into a graph."""

    def __init__(self, device: int = 0):
        self._lib = _lib.load()
        self._ctx = _Context.get(device)
        self._ordinal = device
        h = ctypes.c_void_p()
        _lib.check(self._lib.tmnn_logits_create(self._ctx.handle, ctypes.byref(h)))
        self._h = h

    def close(self) -> None:
        if self._h is not None:
            self._lib.tmnn_logits_destroy(self._h)
            self._h = None

    @property
    def closed(self) -> bool:
        return self._h is None

    def __enter__(self) -> "LogitOps":
        return self

    def __exit__(self, *exc) -> None:
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _run(self, name: str, call: _Call, packed: bytes, stream) -> None:
        if not call.device:
            if stream is not None:
                raise ValueError("stream goes with device tensors")
            _lib.check(getattr(self._lib, name)(self._h, packed))
            return
        if stream is None:
            stream = sys.modules["torch"].cuda.current_stream(self._ordinal).cuda_stream
        elif not isinstance(stream, int):
            stream = stream.cuda_stream
        rc = getattr(self._lib, name + "_device")(self._h, packed, stream)
        if rc:
            _lib.check(rc)

    def _open(self) -> None:
        if self._h is None:
            raise ClosedError("LogitOps is closed")

    # ---- log-probabilities ------------------------------------------------------
    def token_logprobs(self, logits, tokens=None, *, top_k: int = 0, temperature: float = 1.0,
                       out: dict | None = None, stream=None) -> dict:
        """Per row of p = softmax(logits / temperature): `logprob` of the class
        tokens[row] (0 for a negative token, NaN for one >= classes) and its `rank`
        (0: the best; -1 without a token), the `entropy`, the `top_k` best classes
        (`top_ids`, -1 where fewer are not masked, and `top_logprobs`; equal logits go
        to the lower index), and `stats` (largest logit, sum of exp((logits - largest) /
        temperature)), which the backward pass takes.

        `out`: arrays to write to, by these names; it gets those that it lacks, and
        is returned. -inf masks a class; a row whose classes are all masked has log p
        -inf and entropy 0, a row with NaN or +inf gives NaN."""
        self._open()
        c = _Call(logits, "logits", self._ordinal)
        n, v = c.shape
        if not 0 <= top_k <= _lib.LOGITS_MAX_TOP:
            raise ValueError(f"top_k must be in [0, {_lib.LOGITS_MAX_TOP}], got {top_k}")
        out = {} if out is None else out
        tok = _optional(c, tokens, "tokens", (n,), _IDS)
        packed = _PACK_LOGPROBS.pack(
            _SIZE_LOGPROBS, _lib.DTYPES[c.dtype],
            0 if tokens is None else _lib.INDEX_DTYPES[_name(tokens.dtype)], top_k, n, v, c.stride, v,
            c.address(logits), tok, c.output(out, "logprob", (n,), "float32"),
            c.output(out, "entropy", (n,), "float32"), c.output(out, "rank", (n,), "int32"),
            c.output(out, "stats", (n, 2), "float32"),
            c.output(out, "top_ids", (n, top_k), "int32") if top_k else 0,
            c.output(out, "top_logprobs", (n, top_k), "float32") if top_k else 0,
            0, 0, 0, 0, temperature, 0)
        self._run("tmnn_token_logprobs", c, packed, stream)
        return out

    def token_logprobs_backward(self, logits, tokens, forward: dict, *, d_logprob=None,
                                d_entropy=None, d_top_logprobs=None, temperature: float = 1.0,
                                out=None, stream=None):
        """The gradient, in the logits' type, of sum(d_logprob * logprob + d_entropy *
        entropy) + sum(d_top_logprobs * top_logprobs). `forward`: what token_logprobs
        returned for these logits. `out` may be the logits."""
        self._open()
        c = _Call(logits, "logits", self._ordinal)
        n, v = c.shape
        d, d_at, d_stride = c.d_logits(out)
        k = 0
        if d_top_logprobs is not None:
            if len(d_top_logprobs.shape) != 2:
                raise ValueError("d_top_logprobs must be 2D (rows, top_k)")
            k = int(d_top_logprobs.shape[1])
        if d_logprob is not None and tokens is None:
            raise ValueError("d_logprob needs tokens")
        packed = _PACK_LOGPROBS.pack(
            _SIZE_LOGPROBS, _lib.DTYPES[c.dtype],
            0 if tokens is None else _lib.INDEX_DTYPES.get(_name(tokens.dtype), 0), k, n, v, c.stride,
            d_stride, c.address(logits), _optional(c, tokens, "tokens", (n,), _IDS), 0,
            0 if d_entropy is None else c.array(forward["entropy"], "entropy", (n,), _F32), 0,
            c.array(forward["stats"], "stats", (n, 2), _F32),
            c.array(forward["top_ids"], "top_ids", (n, k), _I32) if k else 0, 0,
            _optional(c, d_logprob, "d_logprob", (n,)), _optional(c, d_entropy, "d_entropy", (n,)),
            _optional(c, d_top_logprobs, "d_top_logprobs", (n, k)), d_at, temperature, 0)
        self._run("tmnn_token_logprobs_backward", c, packed, stream)
        return d

    # ---- distillation --------------------------------------------------------------
    @staticmethod
    def _teacher(c: _Call, ids, teacher, kind: str) -> tuple[int, int, int]:
        if kind not in _lib.TEACHER_KINDS:
            raise ValueError(f"kind must be 'logits' or 'logprobs', got {kind!r}")
        if len(ids.shape) != 2:
            raise ValueError("teacher_ids must be 2D (rows, entries)")
        k = int(ids.shape[1])
        n = c.shape[0]
        return (k, c.array(ids, "teacher_ids", (n, k), _IDS),
                c.array(teacher, "teacher", (n, k), _F32))

    def distill(self, logits, teacher_ids, teacher, *, kind: str = "logits",
                temperature: float = 1.0, row_weights=None, gradient: bool = True,
                out: dict | None = None, stream=None) -> dict:
        """Distillation from a teacher's top values: `loss` [rows] =
        row_weights T^2 KL(q || softmax(logits / T)) and, with `gradient`, `d_logits`,
        the gradient of its sum. `kind` "logits": q = softmax(teacher / T) over the
        listed classes; "logprobs": q = exp(teacher), and the classes that are not
        listed count as one class of the remaining mass. Negative ids mark unused
        entries. Rows of weight 0 give 0 and are not read. `stats` [rows, 4] is
        what distill_backward takes.

        `out`: arrays to write to, by these names; it gets those that it lacks, and is
        returned. out["d_logits"] may be the logits."""
        self._open()
        c = _Call(logits, "logits", self._ordinal)
        n, v = c.shape
        out = {} if out is None else out
        k, ids_at, teacher_at = self._teacher(c, teacher_ids, teacher, kind)
        d_at, d_stride = 0, v
        if gradient:
            out["d_logits"], d_at, d_stride = c.d_logits(out.get("d_logits"))
        packed = _PACK_DISTILL.pack(
            _SIZE_DISTILL, _lib.DTYPES[c.dtype], _lib.INDEX_DTYPES[_name(teacher_ids.dtype)],
            _lib.TEACHER_KINDS[kind], n, v, c.stride, d_stride, c.address(logits), ids_at, teacher_at,
            _optional(c, row_weights, "row_weights", (n,)), c.output(out, "loss", (n,), "float32"),
            c.output(out, "stats", (n, 4), "float32", 16), d_at, k, temperature)
        self._run("tmnn_distill", c, packed, stream)
        return out

    def distill_backward(self, logits, teacher_ids, teacher, stats, d_loss, *, kind: str = "logits",
                         temperature: float = 1.0, out=None, stream=None):
        """The gradient, in the logits' type, of sum(d_loss * loss) of an unweighted
        distill call, from its `stats`. `out` may be the logits."""
        self._open()
        c = _Call(logits, "logits", self._ordinal)
        n, v = c.shape
        k, ids_at, teacher_at = self._teacher(c, teacher_ids, teacher, kind)
        d, d_at, d_stride = c.d_logits(out)
        stats_at = c.array(stats, "stats", (n, 4), _F32)
        if stats_at % 16:
            raise ValueError("stats must be 16-byte aligned")
        packed = _PACK_DISTILL.pack(
            _SIZE_DISTILL, _lib.DTYPES[c.dtype], _lib.INDEX_DTYPES[_name(teacher_ids.dtype)],
            _lib.TEACHER_KINDS[kind], n, v, c.stride, d_stride, c.address(logits), ids_at, teacher_at,
            c.array(d_loss, "d_loss", (n,), _F32), 0, stats_at, d_at, k, temperature)
        self._run("tmnn_distill_backward", c, packed, stream)
        return d
