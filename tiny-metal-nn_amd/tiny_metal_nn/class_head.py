"""The class head's calls of LogitOps (include/tmnn_hip.h, class head): operators over
features [rows, dims] and a table of classes [classes, dims], whose class logits are their
products: cross entropy without a tensor of logits and its gradients, logits from 8-bit
operands, and the quantisation that makes these. No counterpart in the reference.

Arrays are looked at as in logits.py: numpy arrays or torch tensors, all of one sort, unit
stride within a row. 8-bit values are torch.float8_e4m3fn tensors or numpy uint8 arrays of the
same bytes, power-of-two scales torch.float8_e8m0fnu or uint8.
"""
from __future__ import annotations

import ctypes
import struct

from . import _lib
from .trainer import DTypeError

# tmnn_class_loss_args, tmnn_class_logits_f8_args (without workspace and its size), tmnn_quantize_f8_args
_PACK_LOSS = struct.Struct("=Iiif7q8Q")
_PACK_LOGITS = struct.Struct("=Iiii6q5Q")
_PACK_WORKSPACE = struct.Struct("=Qq")
_PACK_QUANTIZE = struct.Struct("=Iiii4q3Q")
_SIZE_LOSS, _SIZE_LOGITS = _PACK_LOSS.size + _PACK_WORKSPACE.size, _PACK_LOGITS.size + _PACK_WORKSPACE.size
_NO_WORKSPACE = _PACK_WORKSPACE.pack(0, 0)
_GRADIENTS = {"both": (True, True), "features": (True, False), "table": (False, True), "none": (False, False)}
_BLOCK = 128
_FLOATS = "float32, float16 or bfloat16"


def _matrix(a, x, name: str, codes: dict, want: str, dims: int | None = None) -> tuple[int, int, int, int, int]:
    """(address, row stride, rows, dims, type code) of a matrix; of this width where it is given."""
    if not a.ours(x):
        raise TypeError(f"{name} must be {a.sort}, got {type(x).__name__}")
    code = codes.get(x.dtype)
    if code is None:
        raise DTypeError(f"{name} must be {want}, got {a.name_of(x.dtype)}")
    size = x.shape
    if len(size) != 2:
        raise ValueError(f"{name} must be 2D (rows, dims)")
    rows, width = size
    if width < 1:
        raise ValueError(f"{name} must have at least one value in a row")
    if dims is not None and width != dims:
        raise ValueError(f"{name} must have {dims} values in a row as the features, got {width}")
    at, row, col = a.layout(x, name)
    if rows <= 1:
        row = max(row, width)
    if col != 1 and width > 1 and rows > 0:
        raise ValueError(f"{name} must have unit stride within a row")
    if row < width:
        raise ValueError(f"{name} must have rows that do not overlap")
    return at, row, rows, width, code


class _HeadCalls:
    """What LogitOps has of the class head."""

    def _enqueue(self, a, size_of, on_host, on_device, head: bytes, workspace, stream) -> None:
        """A call whose args are `head` and a workspace: on the device one of the caller's, or memory
        that belongs to the call's stream."""
        if a.device is None:
            if workspace is not None:
                raise ValueError("workspace goes with torch tensors")
            self._run(a, on_host, on_device, head + _NO_WORKSPACE, stream)
            return
        if workspace is None:
            need = ctypes.c_int64()
            rc = size_of(head + _NO_WORKSPACE, ctypes.byref(need))
            if rc:
                _lib.check(rc)
            if need.value == 0:
                self._run(a, on_host, on_device, head + _NO_WORKSPACE, stream)
                return
            if isinstance(stream, int) and stream == -1:
                raise ValueError("the context's own stream needs a workspace of the caller's")
            workspace = a.empty((need.value,), a.torch.uint8)
        elif not a.ours(workspace) or a.name_of(workspace.dtype) != "uint8" or not workspace.is_contiguous():
            raise TypeError("workspace must be a contiguous uint8 tensor")
        else:
            a.place(workspace, "workspace")
        self._run(a, on_host, on_device, head + _PACK_WORKSPACE.pack(workspace.data_ptr(), workspace.numel()), stream)

    def _loss_call(self, a, x, table, labels, temperature, weights, gradient, out, loss, stats, back):
        """(packed args without the workspace, arrays written), for the features and their `x` of _matrix."""
        wanted = _GRADIENTS.get(gradient)
        if wanted is None or (back and gradient == "none"):
            names = "'both', 'features' or 'table'" + ("" if back else " or 'none'")
            raise ValueError(f"gradient must be {names}, got {gradient!r}")
        features, (x, x_row, n, d, code) = x
        if a.ours(table) and table.dtype != features.dtype:
            raise DTypeError(f"table must be {a.name_of(features.dtype)} as the features, "
                             f"got {a.name_of(table.dtype)}")
        y, y_row, v, _, _ = _matrix(a, table, "table", a.float_codes, _FLOATS, d)
        at_labels, index = a.ids(labels, "labels", (n,))
        wrote = [] if back else [out["loss"], out["stats"]]
        grads = [(0, d), (0, d)]
        for i, (name, like) in enumerate((("d_features", features), ("d_table", table))):
            if not wanted[i]:
                continue
            g = out.get(name)
            if g is None:
                g = out[name] = a.empty(tuple(like.shape), like.dtype)
            grads[i] = a.like(g, name, like)
            wrote.append(g)
        head = _PACK_LOSS.pack(_SIZE_LOSS, code, index, temperature, n, v, d, x_row, y_row, grads[0][1], grads[1][1],
                               x, y, at_labels, weights, loss, stats, grads[0][0], grads[1][0])
        return head, wrote

    def class_loss(self, features, table, labels, *, temperature: float = 1.0, row_weights=None,
                   gradient: str = "both", out: dict | None = None, workspace=None, stream=None) -> dict:
        """Softmax cross entropy of the logits features . table / temperature without a tensor
        of them: `loss` [rows] = -row_weights ln p(label) and, by `gradient` ("both", "features",
        "table", "none"), `d_features` and `d_table`, the gradients of its sum. A negative label
        marks a row without one; such rows and those of weight 0 give 0, whatever they hold. A
        label >= classes gives NaN, as do logits that are NaN or +inf and a label's of -inf.
        Classes of probability p have at most 39 + log2 p bits in the gradients (tmnn_hip.h).
        `stats` [rows, 4] is what class_loss_backward takes. temperature: 1e-6 to 1e6.

        `out`: arrays to write to, by these names; it gets those that it lacks, and is
        returned. None may overlap the inputs. `workspace`: a uint8 tensor to work in (with torch
        tensors); the call takes memory of its stream otherwise: about as much as the inputs, up to 256 MB
        of sums in parts for each gradient, and beyond 128 dims 256 MB for a piece of the logits' gradient (or what 256
        classes of all rows take, if that is more), 512 MB for logits if they fit there, and rows * classes / 32
        bytes (/ 16 for few rows)."""
        a = self._arrays(features, stream)
        if out is None:
            out = {}
        x = _matrix(a, features, "features", a.float_codes, _FLOATS)
        rows = (x[2],)
        loss = a.output(out, "loss", rows, a.f32)
        stats = a.output(out, "stats", rows + (4,), a.f32)
        weights = 0 if row_weights is None else a.array(row_weights, "row_weights", rows, a.f32)
        head, wrote = self._loss_call(a, (features, x), table, labels, temperature, weights, gradient, out, loss, stats,
                                      False)
        lib = self._lib
        self._enqueue(a, lambda args, n: lib.tmnn_class_loss_workspace(args, 0, n), lib.tmnn_class_loss,
                      lib.tmnn_class_loss_device, head, workspace, stream)
        a.wrote(wrote)
        return out

    def class_loss_backward(self, features, table, labels, stats, d_loss, *, temperature: float = 1.0,
                            gradient: str = "both", out: dict | None = None, workspace=None,
                            stream=None) -> dict:
        """The gradients of sum(d_loss * loss) of an unweighted class_loss call, from its
        `stats`: `d_features` and `d_table`, by `gradient` ("both", "features", "table")."""
        a = self._arrays(features, stream)
        if out is None:
            out = {}
        x = _matrix(a, features, "features", a.float_codes, _FLOATS)
        rows = (x[2],)
        at_stats = a.array(stats, "stats", rows + (4,), a.f32)
        weights = a.array(d_loss, "d_loss", rows, a.f32)
        head, wrote = self._loss_call(a, (features, x), table, labels, temperature, weights, gradient, out, 0, at_stats,
                                      True)
        lib = self._lib
        self._enqueue(a, lambda args, n: lib.tmnn_class_loss_workspace(args, 1, n), lib.tmnn_class_loss_backward,
                      lib.tmnn_class_loss_backward_device, head, workspace, stream)
        a.wrote(wrote)
        return out

    # ---- 8-bit operands ------------------------------------------------------------
    def class_logits_f8(self, features, feature_scales, table, table_scales, *, dtype="float32", out=None,
                        workspace=None, stream=None):
        """The logits [rows, classes] of e4m3 features [rows, dims] with a scale for each 128 values of
        a row, [rows, ceil(dims / 128)], and an e4m3 table [classes, dims] with one for each
        128 x 128, [ceil(classes / 128), ceil(dims / 128)] (quantize_f8 makes both). Scales are
        float32 or power-of-two bytes (float8_e8m0fnu), alike in both. Logits are `out`, or
        new ones of `dtype`. Rows that start at multiples of 16 bytes, as quantize_f8 lays
        them, are read in place; others are copied in each call."""
        a = self._arrays(features, stream)
        want = "float8_e4m3fn" if a.device is not None else "uint8 (the bytes of e4m3 values)"
        x, x_row, n, d, _ = _matrix(a, features, "features", a.f8_codes, want)
        y, y_row, v, _, _ = _matrix(a, table, "table", a.f8_codes, want, d)
        blocks = -(-d // _BLOCK)
        if not a.ours(feature_scales) or a.scale_codes.get(feature_scales.dtype) is None:
            a.refuse(feature_scales, "feature_scales", (n, blocks), a.scale_names)
        scale = a.scale_codes[feature_scales.dtype]
        sx = a.array(feature_scales, "feature_scales", (n, blocks), feature_scales.dtype)
        sy = a.array(table_scales, "table_scales", (-(-v // _BLOCK), blocks), feature_scales.dtype)
        if out is None:
            out = a.empty((n, v), a.float_type(dtype))
        if not a.ours(out):
            raise TypeError(f"out must be {a.sort}, as the features are, got {type(out).__name__}")
        a.writeable(out, "out")
        if tuple(out.shape) != (n, v):
            raise ValueError(f"out must have shape {(n, v)}, got {tuple(out.shape)}")
        at, row, _, _, code = a.logits(out, "out")
        head = _PACK_LOGITS.pack(_SIZE_LOGITS, code, scale, 0, n, v, d, x_row, y_row, row, x, sx, y, sy, at)
        lib = self._lib
        self._enqueue(a, lib.tmnn_class_logits_f8_workspace, lib.tmnn_class_logits_f8,
                      lib.tmnn_class_logits_f8_device, head, workspace, stream)
        a.wrote([out])
        return out

    def quantize_f8(self, x, *, block_rows: int = 1, scale_dtype="float32", out: dict | None = None,
                    stream=None) -> dict:
        """`values` (e4m3) and `scales` of a matrix: a scale for each block of `block_rows` x 128
        values, 1 for features or 128 for a table; float32 (max |x| / 448) or the power of two at
        or above that (float8_e8m0fnu). What is not finite becomes NaN. New values have rows that
        start at multiples of 16 bytes. `out`: arrays to write to, by these names; it gets
        those that it lacks, and is returned."""
        a = self._arrays(x, stream)
        at, row, n, d, code = _matrix(a, x, "x", a.float_codes, _FLOATS)
        if block_rows not in (1, _BLOCK):
            raise ValueError(f"block_rows must be 1 or {_BLOCK}, got {block_rows}")
        scale = _lib.SCALE_DTYPES.get(a.dtype_name(scale_dtype))
        if scale is None:
            raise DTypeError(f"scale_dtype must be float32 or float8_e8m0fnu, got {scale_dtype}")
        if out is None:
            out = {}
        values = out.get("values")
        if values is None:
            values = out["values"] = a.empty((n, -(-d // 16) * 16), a.f8)[:, :d]
        if not a.ours(values):
            raise TypeError(f"values must be {a.sort}, as x is, got {type(values).__name__}")
        a.writeable(values, "values")
        want = "float8_e4m3fn" if a.device is not None else "uint8"
        to, to_row, rows, _, _ = _matrix(a, values, "values", a.f8_codes, want, d)
        if rows != n:
            raise ValueError(f"values must have shape {(n, d)}, got {tuple(values.shape)}")
        scales = a.output(out, "scales", (-(-n // block_rows), -(-d // _BLOCK)), a.f32 if scale == 0 else a.e8m0)
        self._run(a, self._lib.tmnn_quantize_f8, self._lib.tmnn_quantize_f8_device,
                  _PACK_QUANTIZE.pack(_PACK_QUANTIZE.size, code, scale, block_rows, n, d, row, to_row, at, to, scales),
                  stream)
        a.wrote([values, out["scales"]])
        return out
