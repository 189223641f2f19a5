"""The class-logit operators without a GPU: the C structs against their ctypes
and packed forms, refusals that need no device, and the 64-bit oracle's
gradients against differences of its values."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import logits_oracle as ref

HEADER = Path(__file__).resolve().parent.parent / "include" / "tmnn_hip.h"


def test_struct_layouts_match_the_header(tmp_path):
    from tiny_metal_nn import _lib, logits
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    structs = {"tmnn_token_logprobs_args": (_lib.TokenLogprobsArgs, logits._PACK_LOGPROBS),
               "tmnn_distill_args": (_lib.DistillArgs, logits._PACK_DISTILL)}
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
    for cname, (cls, packed) in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls) == packed.size, cname
        for field, _t in cls._fields_:
            assert int(got[f"{cname}.{field}"]) == getattr(cls, field).offset, (cname, field)
        # the packed form puts its n-th value where the n-th field is
        values = list(range(1, len(cls._fields_) + 1))
        back = cls.from_buffer_copy(packed.pack(*values))
        assert [int(getattr(back, f)) for f, _t in cls._fields_] == values


def test_null_handles_are_rejected_without_a_gpu():
    from tiny_metal_nn import _lib
    lib = _lib.load()
    for name in ("tmnn_token_logprobs", "tmnn_token_logprobs_backward", "tmnn_distill",
                 "tmnn_distill_backward"):
        assert getattr(lib, name)(None, None) == _lib.TMNN_ERR_INVALID_ARGUMENT
        assert b"null" in lib.tmnn_last_error()
        assert getattr(lib, name + "_device")(None, None, None) == _lib.TMNN_ERR_INVALID_ARGUMENT
    out = ctypes.c_void_p()
    assert lib.tmnn_logits_create(None, ctypes.byref(out)) == _lib.TMNN_ERR_INVALID_ARGUMENT
    assert lib.tmnn_logits_destroy(None) == 0


def _differences(f, z, h=1e-5):
    d = np.zeros_like(z)
    for i in np.ndindex(*z.shape):
        up, down = z.copy(), z.copy()
        up[i] += h
        down[i] -= h
        d[i] = (f(up) - f(down)) / (2 * h)
    return d


@pytest.mark.parametrize("t", [0.7, 1.0, 2.0])
def test_oracle_logprob_gradient_against_differences(t):
    rng = np.random.default_rng(3)
    z = rng.normal(size=(3, 7)) * 2
    tokens = np.array([2, -1, 6])
    fwd = ref.token_logprobs(z, tokens, 3, t)
    g, h, gt = rng.normal(size=3), rng.normal(size=3), rng.normal(size=(3, 3))

    def total(x):
        o = ref.token_logprobs(x, tokens, 3, t)
        return (g * o["logprob"]).sum() + (h * o["entropy"]).sum() + (gt * o["top_logprobs"]).sum()

    d, _ = ref.token_logprobs_backward(z, tokens, fwd["top_ids"], g, h, gt, t)
    # second-order differences at h = 1e-5: 1e-10 of the third derivative, 1e-11 of rounding
    assert np.abs(d - _differences(total, z)).max() < 1e-8


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("t", [0.7, 2.0])
def test_oracle_distill_gradient_against_differences(kind, t):
    rng = np.random.default_rng(4)
    z = rng.normal(size=(3, 6)) * 2
    ids = np.array([[0, 3, -1], [5, 1, 5], [2, -1, -1]])  # unused entries, one listed twice
    teacher = rng.normal(size=(3, 3)) * 1.5
    if kind == "logprobs":
        teacher = teacher - 4.0
    w = np.array([0.5, 1.0, 2.0])
    _, d, _, _ = ref.distill(z, ids, teacher, kind, t, w)
    diff = _differences(lambda x: ref.distill(x, ids, teacher, kind, t, w)[0].sum(), z)
    assert np.abs(d - diff).max() < 1e-8


def test_host_outputs_must_be_writeable():
    """A mapped read-only array would fault where the copy out writes to it."""
    from tiny_metal_nn import logits
    arrays = logits._HostArrays()
    z = np.zeros((2, 3), np.float32)
    fixed, free = np.zeros((2, 3), np.float32), np.zeros((2, 3), np.float32)
    fixed.setflags(write=False)
    assert arrays.output({"loss": free[0]}, "loss", (3,), np.float32) == free.ctypes.data
    with pytest.raises(ValueError, match="loss must be writeable"):
        arrays.output({"loss": fixed[0]}, "loss", (3,), np.float32)
    assert arrays.like(free, "d_logits", z) == (free.ctypes.data, 3)
    with pytest.raises(ValueError, match="d_logits must be writeable"):
        arrays.like(fixed, "d_logits", z)
    # what is only read need not be
    assert arrays.logits(fixed, "logits")[0] == fixed.ctypes.data
