"""The class head without a GPU: the C structs against their ctypes and packed forms,
refusals that need no device, workspace sizes, and the 64-bit oracle's gradients against
differences of its values."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import head_oracle as ref  # noqa: E402

HEADER = Path(__file__).resolve().parent.parent / "include" / "tmnn_hip.h"


def test_struct_layouts_match_the_header(tmp_path):
    from tiny_metal_nn import _lib, class_head
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    tail = class_head._PACK_WORKSPACE
    structs = {"tmnn_class_loss_args": (_lib.ClassLossArgs, (class_head._PACK_LOSS, tail)),
               "tmnn_class_logits_f8_args": (_lib.ClassLogitsF8Args, (class_head._PACK_LOGITS, tail)),
               "tmnn_quantize_f8_args": (_lib.QuantizeF8Args, (class_head._PACK_QUANTIZE,))}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "tmnn_hip.h"', "int main(void) {"]
    for cname, (cls, _) in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        for field, _t in cls._fields_:
            lines.append(f'printf("{cname}.{field} %zu\\n", offsetof({cname}, {field}));')
    lines.append("return 0; }")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run([cc, "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    got = dict(line.rsplit(" ", 1) for line in
               subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cname, (cls, packs) in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls) == sum(p.size for p in packs), cname
        for field, _t in cls._fields_:
            assert int(got[f"{cname}.{field}"]) == getattr(cls, field).offset, (cname, field)
        # the packed form puts its n-th value where the n-th field is
        values = list(range(1, len(cls._fields_) + 1))
        packed, at = b"", 0
        for p in packs:
            count = len(p.unpack(bytes(p.size)))
            packed += p.pack(*values[at:at + count])
            at += count
        back = cls.from_buffer_copy(packed)
        assert [int(getattr(back, f)) for f, _t in cls._fields_] == values


def test_null_handles_are_rejected_without_a_gpu():
    from tiny_metal_nn import _lib
    lib = _lib.load()
    for name in ("tmnn_class_loss", "tmnn_class_loss_backward", "tmnn_class_logits_f8", "tmnn_quantize_f8"):
        assert getattr(lib, name)(None, None) == _lib.TMNN_ERR_INVALID_ARGUMENT
        assert b"null" in lib.tmnn_last_error()
        assert getattr(lib, name + "_device")(None, None, None) == _lib.TMNN_ERR_INVALID_ARGUMENT


def loss_args(**more):
    from tiny_metal_nn import _lib
    a = _lib.ClassLossArgs(ctypes.sizeof(_lib.ClassLossArgs), 0, 0, 1.0, 8, 5, 7, 7, 7, 7, 7)
    for k, v in more.items():
        setattr(a, k, v)
    return bytes(a)


def logits_args(**more):
    from tiny_metal_nn import _lib
    a = _lib.ClassLogitsF8Args(ctypes.sizeof(_lib.ClassLogitsF8Args), 0, 0, 0, 8, 5, 7, 7, 7, 5)
    for k, v in more.items():
        setattr(a, k, v)
    return bytes(a)


@pytest.mark.parametrize("bad,frag", [
    ({"struct_size": 8}, "struct_size"), ({"dtype": 3}, "dtype"), ({"index_dtype": 2}, "index_dtype"),
    ({"temperature": 0.0}, "temperature"), ({"temperature": float("nan")}, "temperature"), ({"rows": -1}, "rows"),
    ({"rows": 1 << 25}, "rows"), ({"classes": 0}, "classes"), ({"classes": (1 << 24) + 1}, "classes"),
    ({"dims": 0}, "dims"), ({"dims": 1 << 17}, "dims"), ({"rows": 1 << 20, "classes": 1 << 20}, "rows x classes"),
    ({"feature_stride": 6}, "stride"), ({"table_stride": 6}, "stride"),
    ({"d_features": 64, "d_feature_stride": 6}, "d_feature_stride"), ({"d_table": 64, "d_table_stride": 6}, "d_table_stride"),
])
def test_loss_workspace_refuses(bad, frag):
    from tiny_metal_nn import _lib
    lib, n = _lib.load(), ctypes.c_int64(7)
    for back in (0, 1):
        assert lib.tmnn_class_loss_workspace(loss_args(**bad), back, ctypes.byref(n)) == _lib.TMNN_ERR_INVALID_ARGUMENT
        assert frag.encode() in lib.tmnn_last_error() and n.value == 0
    assert lib.tmnn_class_loss_workspace(loss_args(), 0, None) == _lib.TMNN_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("bad,frag", [
    ({"struct_size": 8}, "struct_size"), ({"dtype": 3}, "dtype"), ({"scale_dtype": 2}, "scale_dtype"),
    ({"rows": -1}, "rows"), ({"classes": 0}, "classes"), ({"dims": 0}, "dims"), ({"feature_stride": 6}, "stride"),
    ({"table_stride": 6}, "stride"), ({"logit_stride": 4}, "logit_stride"),
])
def test_logits_workspace_refuses(bad, frag):
    from tiny_metal_nn import _lib
    lib, n = _lib.load(), ctypes.c_int64(7)
    assert lib.tmnn_class_logits_f8_workspace(logits_args(**bad), ctypes.byref(n)) == _lib.TMNN_ERR_INVALID_ARGUMENT
    assert frag.encode() in lib.tmnn_last_error() and n.value == 0


def workspace(**args):
    from tiny_metal_nn import _lib
    lib, n = _lib.load(), ctypes.c_int64()
    assert lib.tmnn_class_loss_workspace(loss_args(**args), 0, ctypes.byref(n)) == 0
    return n.value


def test_workspace_sizes():
    """The logits are not in the workspace; without rows, and for 8-bit operands that lie at multiples of 16
    bytes, none is needed."""
    from tiny_metal_nn import _lib
    n, d, v = 4096, 2048, 131072
    big = dict(dtype=2, rows=n, classes=v, dims=d, feature_stride=d, table_stride=d, d_feature_stride=d,
               d_table_stride=d, features=256, table=512)
    assert workspace(**big) < 64 << 20  # sums of a row's tiles, nothing laid out
    both = workspace(**big, d_features=1024, d_table=2048)
    # the table and the features once each (and weighted), d of a piece, sums of d_features
    assert both < 2 * (v + 2 * n) * d + (300 << 20) + 4 * n * d * 4 < n * v * 4
    assert workspace(rows=0) == 0
    lib, got = _lib.load(), ctypes.c_int64(7)
    args = logits_args(rows=512, classes=65536, dims=1000, feature_stride=1008, table_stride=1008, logit_stride=65536,
                       features=256, table=512)
    assert lib.tmnn_class_logits_f8_workspace(args, ctypes.byref(got)) == 0 and got.value == 0
    args = logits_args(rows=512, classes=65536, dims=1000, feature_stride=1008, table_stride=1000, logit_stride=65536,
                       features=256, table=512)
    assert lib.tmnn_class_logits_f8_workspace(args, ctypes.byref(got)) == 0 and 65536 * 1008 <= got.value < 65536 * 1024


@pytest.mark.parametrize("t", [0.3, 1.0, 2.0])
def test_oracle_gradient_against_differences(t):
    g = torch.Generator().manual_seed(4)
    h = torch.randn(5, 6, generator=g, dtype=torch.float64)
    w = torch.randn(7, 6, generator=g, dtype=torch.float64)
    labels = torch.tensor([2, -1, 6, 0, 3])
    weights = torch.tensor([0.5, 1.0, -2.0, 1.0, 0.0], dtype=torch.float64)
    got = ref.class_loss(h, w, labels, weights, t)
    for name, x in (("d_features", h), ("d_table", w)):
        for i in np.ndindex(*x.shape):
            step = 1e-5
            keep = x[i].item()
            x[i] = keep + step
            up = ref.class_loss(h, w, labels, weights, t)["loss"].sum()
            x[i] = keep - step
            down = ref.class_loss(h, w, labels, weights, t)["loss"].sum()
            x[i] = keep
            # second-order differences: 1e-10 of the third derivative (below 100 / t^3 here), 1e-11 of rounding
            assert abs((up - down) / (2 * step) - got[name][i]) < 1e-8 / t ** 3


def test_oracle_quantisation_is_the_nearest():
    x = torch.randn(3, 300, generator=torch.Generator().manual_seed(2)) * 5
    for power in (False, True):
        values, scales = ref.quantize(x, 1, power)
        y = x.double() / ref.spread(scales, 3, 300, 1)
        grid = torch.cat([-ref.GRID, ref.GRID])
        nearest = (y.unsqueeze(2) - grid).abs().amin(2)
        assert torch.equal((y - values).abs(), nearest)
        assert (values.abs().amax() == 448.0) or power


def test_host_arrays_are_checked_before_any_call():
    """Shapes, types and strides of numpy arrays, by the checks that every call shares."""
    from tiny_metal_nn import DTypeError, class_head, logits
    a = logits._HostArrays()
    x = np.zeros((3, 5), np.float32)
    assert class_head._matrix(a, x, "x", a.float_codes, "float32")[1:] == (5, 3, 5, 0)
    assert class_head._matrix(a, x[:, :2], "x", a.float_codes, "float32")[1:] == (5, 3, 2, 0)
    for bad, error, frag in ((x.tolist(), TypeError, "numpy"), (x.astype(np.int32), DTypeError, "float32"),
                             (x[0], ValueError, "2D"), (x[:, :0], ValueError, "at least one"),
                             (x.T, ValueError, "unit stride"), (x[::-1], ValueError, "overlap")):
        with pytest.raises(error, match=frag):
            class_head._matrix(a, bad, "x", a.float_codes, "float32")
    with pytest.raises(ValueError, match="4 values in a row"):
        class_head._matrix(a, x, "x", a.float_codes, "float32", 4)
