"""LogitOps: operators over rows of class logits (include/tmnn_hip.h, class
logits): log-probabilities of given classes with rank, entropy and the best
alternatives, their gradient, and distillation from a teacher's top values.

Arrays are numpy arrays (copied in and out; the results are there on return) or
torch tensors of the operators' device (the call is only enqueued, on torch's
current stream unless `stream` says otherwise; arrays that a call makes belong to its
stream). All arrays of a call are of one sort. Logits are float32, float16 or (tensors)
bfloat16, [rows, classes] with unit stride within a row; class ids int32 or int64;
everything else float32 / int32 and contiguous. No counterpart in the reference.

The calls are no part of torch's autograd: results have no history, whether or not the
logits require gradients, and a loss's gradient is the *_backward calls' (in a
torch.autograd.Function, or passed to logits.backward()). Tensors that a call writes to are
marked as changed in place, so that autograd refuses a backward pass that saved their old values.
"""
from __future__ import annotations

import copy
import ctypes
import struct
import sys

import numpy as np

from . import _lib
from .class_head import _HeadCalls
from .trainer import ClosedError, DTypeError, _Context

# tmnn_token_logprobs_args, tmnn_distill_args
_PACK_LOGPROBS = struct.Struct("=Iiii4q12Qfi")
_PACK_DISTILL = struct.Struct("=Iiii4q7Qif")
_FORWARD = ("logprob", "entropy", "rank", "stats")
_FORWARD_TOP = _FORWARD + ("top_ids", "top_logprobs")
_SIZE_LOGPROBS, _SIZE_DISTILL = _PACK_LOGPROBS.size, _PACK_DISTILL.size


class _Arrays:
    """How the arrays of a call are looked at: numpy's, or torch's on a device.
    Small calls are bound by this host work, so what is right passes in one
    expression and only what is not is looked at closely."""

    def __init__(self, lib, sort: str):
        self.sort = sort
        self.f32, self.i32 = getattr(lib, "float32"), getattr(lib, "int32")

    def name_of(self, dtype) -> str:
        return str(dtype).replace("torch.", "")

    def refuse(self, x, name: str, shape: tuple, want: str):
        if not self.ours(x):
            raise TypeError(f"{name} must be {self.sort}, as the logits are, got {type(x).__name__}")
        if self.name_of(x.dtype) not in want.split(" or "):
            raise DTypeError(f"{name} must be {want}, got {self.name_of(x.dtype)}")
        if tuple(x.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")

    def logits(self, x, name: str, shape: tuple | None = None, dtype=None) -> tuple:
        """(address, row stride, rows, classes, type code) of a matrix; of this shape
        and type where they are given."""
        code = self.float_codes.get(x.dtype)
        if code is None or (dtype is not None and x.dtype != dtype):
            want = "float32, float16 or bfloat16" if dtype is None else f"{self.name_of(dtype)} as the logits"
            raise DTypeError(f"{name} must be {want}, got {self.name_of(x.dtype)}")
        size = x.shape
        if len(size) != 2:
            raise ValueError(f"{name} must be 2D (rows, classes)")
        if shape is not None and size != shape:
            raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(size)}")
        rows, classes = size
        at, row, col = self.layout(x, name)
        if classes < 1:
            raise ValueError(f"{name} must have at least one class")
        if rows <= 1:
            row = max(row, classes)
        if col != 1 and classes > 1 and rows > 0:
            raise ValueError(f"{name} must have unit stride within a row")
        if row < classes:
            raise ValueError(f"{name} must have rows that do not overlap")
        return at, row, rows, classes, code

    def like(self, x, name: str, logits) -> tuple[int, int]:
        """Address and row stride of a matrix to write to, like the logits."""
        if not self.ours(x):
            raise TypeError(f"{name} must be {self.sort}, as the logits are, got {type(x).__name__}")
        self.writeable(x, name)
        return self.logits(x, name, logits.shape, logits.dtype)[:2]

    def ids(self, x, name: str, shape: tuple) -> tuple[int, int]:
        """Address and type code of class ids."""
        if self.ours(x):
            code = self.index_codes.get(x.dtype)
            if code is not None:
                return self.array(x, name, shape, x.dtype), code
        self.refuse(x, name, shape, "int32 or int64")

    def output(self, out: dict, key: str, shape: tuple, dtype) -> int:
        x = out.get(key)
        if x is None:
            x = out[key] = self.empty(shape, dtype)
        at = self.array(x, key, shape, dtype)
        self.writeable(x, key)
        return at

    def writeable(self, x, name: str) -> None:
        pass

    def dtype_name(self, dtype) -> str:
        """A type's name, given as a type of the library's or by name."""
        return dtype if isinstance(dtype, str) else self.name_of(dtype)

    def float_type(self, dtype):
        name = self.dtype_name(dtype)
        for t in self.float_codes:
            if self.name_of(t) == name:
                return t
        raise DTypeError(f"dtype must be float32, float16 or bfloat16, got {name}")

    def wrote(self, arrays: list) -> None:
        """After a call: what it has written to."""


class _HostArrays(_Arrays):
    device = None

    def __init__(self):
        super().__init__(np, "a numpy array")
        self.float_codes = {np.dtype(k): c for k, c in _lib.DTYPES.items() if k != "bfloat16"}
        self.index_codes = {np.dtype(k): c for k, c in _lib.INDEX_DTYPES.items()}
        # numpy has no 8-bit floating point: its bytes
        self.f8 = self.e8m0 = np.uint8
        self.f8_codes = {np.dtype(np.uint8): 0}
        self.scale_codes = {np.dtype(np.float32): 0, np.dtype(np.uint8): 1}
        self.scale_names = "float32 or uint8"

    def dtype_name(self, dtype) -> str:
        return dtype if isinstance(dtype, str) else np.dtype(dtype).name

    @staticmethod
    def ours(x) -> bool:
        return isinstance(x, np.ndarray)

    def array(self, x, name: str, shape: tuple, dtype) -> int:
        if not (self.ours(x) and x.dtype == dtype and x.shape == shape):
            self.refuse(x, name, shape, np.dtype(dtype).name)
        if not x.flags.c_contiguous:
            raise ValueError(f"{name} must be contiguous")
        return x.ctypes.data

    @staticmethod
    def layout(x, name: str) -> tuple[int, int, int]:
        size = x.itemsize
        row, col = (s // size if s % size == 0 else -1 for s in x.strides)
        return x.ctypes.data, row, col

    def writeable(self, x, name: str) -> None:
        if not x.flags.writeable:
            raise ValueError(f"{name} must be writeable")

    @staticmethod
    def empty(shape: tuple, dtype):
        return np.empty(shape, dtype)


class _DeviceArrays(_Arrays):
    def __init__(self, torch, device: int):
        super().__init__(torch, "a torch tensor")
        self.torch, self.device = torch, device
        self.float_codes = {getattr(torch, k): c for k, c in _lib.DTYPES.items()}
        self.index_codes = {getattr(torch, k): c for k, c in _lib.INDEX_DTYPES.items()}
        self.f8, self.e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
        self.f8_codes = {self.f8: 0}
        self.scale_codes = {getattr(torch, k): c for k, c in _lib.SCALE_DTYPES.items()}
        self.scale_names = " or ".join(_lib.SCALE_DTYPES)
        self.raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda d: torch.cuda.current_stream(d).cuda_stream)
        self.side = None  # the stream that new arrays belong to, if not the current one
        self.wrote = torch.autograd.graph.increment_version

    def on(self, stream) -> "_DeviceArrays":
        """The same for a call on a stream of the caller's. Its new arrays are of that
        stream's memory: memory that the current stream has freed may still be in use there."""
        cuda = self.torch.cuda
        if isinstance(stream, int):
            if stream == -1:  # the context's own (TMNN_STREAM_CONTEXT): torch has none of its memory
                return self
            stream = cuda.ExternalStream(stream, self.device)
        a = copy.copy(self)
        a.side = stream
        return a

    @staticmethod
    def ours(x) -> bool:
        return hasattr(x, "data_ptr")

    def place(self, x, name: str) -> None:
        if x.get_device() != self.device:
            raise ValueError(f"{name} must be on device {self.device}, is on {x.device}")

    def array(self, x, name: str, shape: tuple, dtype) -> int:
        try:
            if (x.dtype is dtype and x.shape == shape and x.get_device() == self.device
                    and x.is_contiguous()):
                return x.data_ptr()
        except AttributeError:
            pass
        self.refuse(x, name, shape, self.name_of(dtype))
        self.place(x, name)
        raise ValueError(f"{name} must be contiguous")

    def output(self, out: dict, key: str, shape: tuple, dtype) -> int:
        x = out.get(key)
        if x is None:
            x = out[key] = self.empty(shape, dtype)
            return x.data_ptr()
        try:  # (as in `array`, without its call)
            if (x.dtype is dtype and x.shape == shape and x.get_device() == self.device
                    and x.is_contiguous()):
                return x.data_ptr()
        except AttributeError:
            pass
        return self.array(x, key, shape, dtype)

    def layout(self, x, name: str) -> tuple[int, int, int]:
        if x.get_device() != self.device:
            self.place(x, name)
        return (x.data_ptr(), *x.stride())

    def empty(self, shape: tuple, dtype):
        if self.side is None:
            return self.torch.empty(shape, dtype=dtype, device=f"cuda:{self.device}")
        with self.torch.cuda.stream(self.side):
            return self.torch.empty(shape, dtype=dtype, device=f"cuda:{self.device}")


class LogitOps(_HeadCalls):
    """Operators over rows of class logits, and over features and a table of classes
    (class_head.py), on one device.

    Holds the workspace of its calls: calls through one object are ordered where
    they share it, also across streams. Use one object per thread, and one of its
    own for a stream that is captured into a graph."""

    def __init__(self, device: int = 0):
        lib = self._lib = _lib.load()
        self._ctx = _Context.get(device)
        self._ordinal = device
        h = ctypes.c_void_p()
        _lib.check(lib.tmnn_logits_create(self._ctx.handle, ctypes.byref(h)))
        self._h = h
        self._host = _HostArrays()
        self._device: _DeviceArrays | None = None

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

    def _arrays(self, logits, stream) -> _Arrays:
        if self._h is None:
            raise ClosedError("LogitOps is closed")
        if isinstance(logits, np.ndarray):
            if stream is not None:
                raise ValueError("stream goes with torch tensors")
            return self._host
        if self._device is None:
            torch = sys.modules.get("torch")
            if torch is None or not isinstance(logits, torch.Tensor):
                raise TypeError(f"logits must be a numpy array or a torch tensor, got {type(logits).__name__}")
            self._device = _DeviceArrays(torch, self._ordinal)
        elif not hasattr(logits, "data_ptr"):
            raise TypeError(f"logits must be a numpy array or a torch tensor, got {type(logits).__name__}")
        return self._device if stream is None else self._device.on(stream)

    def _run(self, a: _Arrays, on_host, on_device, packed: bytes, stream) -> None:
        if a.device is None:
            rc = on_host(self._h, packed)
        else:
            if stream is None:
                stream = a.raw_stream(a.device)
            elif not isinstance(stream, int):
                stream = stream.cuda_stream
            rc = on_device(self._h, packed, stream)
        if rc:
            _lib.check(rc)

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
        a = self._arrays(logits, stream)
        at, stride, n, v, code = a.logits(logits, "logits")
        if not 0 <= top_k <= _lib.LOGITS_MAX_TOP:
            raise ValueError(f"top_k must be in [0, {_lib.LOGITS_MAX_TOP}], got {top_k}")
        if out is None:
            out = {}
        rows = (n,)
        tok, index = (0, 0) if tokens is None else a.ids(tokens, "tokens", rows)
        f32, i32 = a.f32, a.i32
        ids = best = 0
        if top_k:
            ids = a.output(out, "top_ids", (n, top_k), i32)
            best = a.output(out, "top_logprobs", (n, top_k), f32)
        self._run(a, self._lib.tmnn_token_logprobs, self._lib.tmnn_token_logprobs_device,
                  _PACK_LOGPROBS.pack(
                      _SIZE_LOGPROBS, code, index, top_k, n, v, stride, v, at, tok,
                      a.output(out, "logprob", rows, f32), a.output(out, "entropy", rows, f32),
                      a.output(out, "rank", rows, i32), a.output(out, "stats", (n, 2), f32),
                      ids, best, 0, 0, 0, 0, temperature, 0), stream)
        a.wrote([out[name] for name in (_FORWARD_TOP if top_k else _FORWARD)])
        return out

    def token_logprobs_backward(self, logits, tokens, forward: dict, *, d_logprob=None,
                                d_entropy=None, d_top_logprobs=None, temperature: float = 1.0,
                                out=None, stream=None):
        """The gradient, in the logits' type, of sum(d_logprob * logprob + d_entropy *
        entropy) + sum(d_top_logprobs * top_logprobs). `forward`: what token_logprobs
        returned for these logits. `out` may be the logits."""
        a = self._arrays(logits, stream)
        at, stride, n, v, code = a.logits(logits, "logits")
        if out is None:
            out = a.empty(logits.shape, logits.dtype)
        d_at, d_stride = a.like(out, "d_logits", logits)
        rows, f32 = (n,), a.f32
        tok, index = (0, 0) if tokens is None else a.ids(tokens, "tokens", rows)
        k = ids = g_token = g_entropy = entropy = g_top = 0
        if d_logprob is not None:
            if tokens is None:
                raise ValueError("d_logprob needs tokens")
            g_token = a.array(d_logprob, "d_logprob", rows, f32)
        if d_entropy is not None:
            g_entropy = a.array(d_entropy, "d_entropy", rows, f32)
            entropy = a.array(forward["entropy"], "entropy", rows, f32)
        if d_top_logprobs is not None:
            if len(d_top_logprobs.shape) != 2:
                raise ValueError("d_top_logprobs must be 2D (rows, top_k)")
            k = int(d_top_logprobs.shape[1])
            if k:
                g_top = a.array(d_top_logprobs, "d_top_logprobs", (n, k), f32)
                ids = a.array(forward["top_ids"], "top_ids", (n, k), a.i32)
        self._run(a, self._lib.tmnn_token_logprobs_backward,
                  self._lib.tmnn_token_logprobs_backward_device,
                  _PACK_LOGPROBS.pack(
                      _SIZE_LOGPROBS, code, index, k, n, v, stride, d_stride, at, tok, 0, entropy, 0,
                      a.array(forward["stats"], "stats", (n, 2), f32), ids, 0, g_token, g_entropy,
                      g_top, d_at, temperature, 0), stream)
        a.wrote([out])
        return out

    # ---- distillation --------------------------------------------------------------
    @staticmethod
    def _teacher(a: _Arrays, n: int, ids, teacher, kind: str) -> tuple[int, int, int, int, int]:
        code = _lib.TEACHER_KINDS.get(kind)
        if code is None:
            raise ValueError(f"kind must be 'logits' or 'logprobs', got {kind!r}")
        if len(ids.shape) != 2:
            raise ValueError("teacher_ids must be 2D (rows, entries)")
        k = int(ids.shape[1])
        at, index = a.ids(ids, "teacher_ids", (n, k))
        return code, k, at, index, a.array(teacher, "teacher", (n, k), a.f32)

    def distill(self, logits, teacher_ids, teacher, *, kind: str = "logits",
                temperature: float = 1.0, row_weights=None, gradient: bool = True,
                out: dict | None = None, stream=None) -> dict:
        """Distillation from a teacher's top values: `loss` [rows] =
        row_weights T^2 KL(q || softmax(logits / T)) and, with `gradient`, `d_logits`,
        the gradient of its sum. `kind` "logits": q = softmax(teacher / T) over the
        listed classes; "logprobs": q = exp(teacher), and the classes that are not
        listed count as one class of the remaining mass. Negative ids mark unused
        entries. Rows of weight 0 give 0, whatever they hold. `stats` [rows, 4] is
        what distill_backward takes.

        `out`: arrays to write to, by these names; it gets those that it lacks, and is
        returned. out["d_logits"] may be the logits."""
        a = self._arrays(logits, stream)
        at, stride, n, v, code = a.logits(logits, "logits")
        if out is None:
            out = {}
        kind_code, k, ids, index, values = self._teacher(a, n, teacher_ids, teacher, kind)
        d_at, d_stride = 0, v
        if gradient:
            d = out.get("d_logits")
            if d is None:
                d = out["d_logits"] = a.empty(logits.shape, logits.dtype)
            d_at, d_stride = a.like(d, "d_logits", logits)
        f32 = a.f32
        self._run(a, self._lib.tmnn_distill, self._lib.tmnn_distill_device,
                  _PACK_DISTILL.pack(
                      _SIZE_DISTILL, code, index, kind_code, n, v, stride, d_stride, at, ids, values,
                      0 if row_weights is None else a.array(row_weights, "row_weights", (n,), f32),
                      a.output(out, "loss", (n,), f32), a.output(out, "stats", (n, 4), f32), d_at, k,
                      temperature), stream)
        a.wrote([out["loss"], out["stats"], out["d_logits"]] if gradient else [out["loss"], out["stats"]])
        return out

    def distill_backward(self, logits, teacher_ids, teacher, stats, d_loss, *, kind: str = "logits",
                         temperature: float = 1.0, out=None, stream=None):
        """The gradient, in the logits' type, of sum(d_loss * loss) of an unweighted
        distill call, from its `stats`. `out` may be the logits."""
        a = self._arrays(logits, stream)
        at, stride, n, v, code = a.logits(logits, "logits")
        kind_code, k, ids, index, values = self._teacher(a, n, teacher_ids, teacher, kind)
        if out is None:
            out = a.empty(logits.shape, logits.dtype)
        d_at, d_stride = a.like(out, "d_logits", logits)
        self._run(a, self._lib.tmnn_distill_backward, self._lib.tmnn_distill_backward_device,
                  _PACK_DISTILL.pack(
                      _SIZE_DISTILL, code, index, kind_code, n, v, stride, d_stride, at, ids, values,
                      a.array(d_loss, "d_loss", (n,), a.f32), 0, a.array(stats, "stats", (n, 4), a.f32),
                      d_at, k, temperature), stream)
        a.wrote([out])
        return out
