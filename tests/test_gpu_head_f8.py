"""Logits from 8-bit operands and the quantisation that makes them, on the GPU
against 64 bits (head_oracle.py). Marked gpu.

Tolerances, with u = 2^-24: products of e4m3 values are exact in fp32, a logit is
their sum in fp32, with one scaling more for each block of 128: (D + D / 128) u of the
sum of absolute terms and one rounding of the products of scales for fp32 scales (4 u), then
half an ulp of the logits' type. 16-bit logits may be summed by an instruction that adds eight
products at a time, each cut to 2^-13 of the largest of the eight (its exponent): 7 2^-13 of the
largest, which is at most the sum of the eight's magnitudes. Quantised values and scales are exact: the nearest values."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import head_oracle as ref  # noqa: E402
from test_gpu_class_loss import DEV, HALF_ULP, TYPES, U, matrix, ops  # noqa: E402,F401

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
SCALES = {"f32": torch.float32, "e8m0": E8M0}


def quantities(n, d, g, wide=True):
    x = torch.randn(n, d, device=DEV, generator=g)
    return x * torch.exp(2 * torch.randn(d, device=DEV, generator=g)) if wide else x


def same(got, want):
    got, want = got.float().double().cpu(), want.double().cpu()
    assert ((got == want) | (got.isnan() & want.isnan())).all(), (got != want).nonzero()[:5]


@pytest.mark.parametrize("scale", list(SCALES))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (1, 127), (3, 128), (5, 129), (130, 300), (257, 1000), (128, 256)],
                         ids=lambda s: "x".join(map(str, s)))
def test_quantize(ops, shape, block_rows, dtype, scale):
    g = torch.Generator(device=DEV).manual_seed(sum(shape))
    x = matrix(quantities(*shape, g), dtype, pad=shape[0] % 3, offset=shape[1] % 2)
    got = ops.quantize_f8(x, block_rows=block_rows, scale_dtype=SCALES[scale])
    values, scales = ref.quantize(x, block_rows, scale == "e8m0")
    same(got["scales"], scales)
    same(got["values"], values)
    assert got["values"].stride(0) % 16 == 0


@pytest.mark.parametrize("scale", list(SCALES))
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_odd_blocks(ops, block_rows, scale):
    """Zeros, one value alone, values on the borders between two e4m3 numbers, tiny and huge
    blocks, NaN and infinities."""
    x = torch.zeros(7 * 128, 256)
    x[128, 5] = -3.0
    # 448 and the middles of all neighbours: quotients that end on a border, times odd scales
    mid = ((ref.GRID[1:] + ref.GRID[:-1]) / 2).float()
    for r in range(128):
        x[256 + r, :126] = mid * (1 + r / 128)
        x[256 + r, 126] = 448.0 * (1 + r / 128)
    x[384:512] = torch.randn(128, 256) * 1e-38
    x[512:640] = torch.randn(128, 256) * 1e37
    x[640:768] = torch.randn(128, 256)
    x[640, 3], x[641, 4], x[642, 5] = float("nan"), float("inf"), -float("inf")
    x[768, :] = float("nan")
    x = x.to(DEV)
    got = ops.quantize_f8(x, block_rows=block_rows, scale_dtype=SCALES[scale])
    values, scales = ref.quantize(x, block_rows, scale == "e8m0")
    same(got["scales"], scales)
    same(got["values"], values)


def operands(n, d, v, scale, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x, w = quantities(n, d, g, False), quantities(v, d, g, False)
    out = []
    for m, rows in ((x, 1), (w, 128)):
        q, s = ref.quantize(m, rows, scale == "e8m0")
        out += [q.float().to(E4M3).to(DEV), s.to(SCALES[scale]).to(DEV)]
    return out


def laid(q, to=16):
    """Rows that start at multiples of `to` bytes, what lies between them being NaN."""
    n, d = q.shape
    place = torch.full((n, -(-d // to) * to), 255, device=DEV, dtype=torch.uint8)
    place[:, :d] = q.view(torch.uint8)
    return place.view(E4M3)[:, :d]


def check_logits(got, x, sx, w, sw, dtype):
    want, size = ref.logits_f8(x, sx, w, sw)
    d = x.shape[1]
    rel, step = HALF_ULP[dtype]
    err = size * ((d + d / 128 + 4) * U + (0.0 if dtype == "f32" else 7 * 2.0 ** -13))
    err = err + rel * (want.abs() + err) + step
    bad = ~((got.double() - want).abs() <= err + 1e-30)
    assert not bad.any(), (bad.nonzero()[:5], ((got.double() - want).abs() / err).max())


@pytest.mark.parametrize("scale", list(SCALES))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 16, 3), (3, 127, 5), (17, 128, 129), (64, 129, 300), (130, 1000, 257),
                                   (1, 1024, 5003), (33, 2050, 70), (300, 48, 1000), (2, 4096, 100), (1030, 640, 2300)],
                         ids=lambda s: "x".join(map(str, s)))
def test_logits(ops, shape, dtype, scale):
    n, d, v = shape
    x, sx, w, sw = operands(n, d, v, scale, n + d + v)
    got = ops.class_logits_f8(laid(x), sx, laid(w), sw, dtype=TYPES[dtype])
    assert got.dtype == TYPES[dtype] and got.shape == (n, v)
    check_logits(got, x, sx, w, sw, dtype)
    # rows at other places give the same bits, into a matrix of another stride too
    out = matrix(torch.zeros(n, v, device=DEV), dtype, pad=3, offset=1)
    ops.class_logits_f8(x, sx, laid(w, 32), sw, out=out)
    assert torch.equal(out, got)


@pytest.mark.parametrize("scale", list(SCALES))
def test_logits_large(ops, scale):
    x, sx, w, sw = operands(2050, 1152, 9001, scale, 3)
    check_logits(ops.class_logits_f8(laid(x), sx, laid(w), sw, dtype="bfloat16"), x, sx, w, sw, "bf16")


@pytest.mark.parametrize("scale", list(SCALES))
def test_logits_of_nan(ops, scale):
    """A NaN value or scale stays within its rows, its classes and their block."""
    x, sx, w, sw = operands(40, 300, 300, scale, 8)
    bits = x.view(torch.uint8)
    bits[3, 299] = 0x7f
    w.view(torch.uint8)[7, 0] = 0xff
    if scale == "f32":
        sx[11, 1] = float("nan")
        sw[2, 2] = float("nan")
    else:
        sx.view(torch.uint8)[11, 1] = 255
        sw.view(torch.uint8)[2, 2] = 255
    got = ops.class_logits_f8(laid(x), sx, laid(w), sw)
    nan = torch.zeros(40, 300, dtype=torch.bool, device=DEV)
    nan[3], nan[11], nan[:, 7], nan[:, 256:] = True, True, True, True
    assert torch.equal(got.isnan(), nan)
    clean = [t.clone() for t in (x, w)]
    want = ops.class_logits_f8(laid(clean[0]), torch.nan_to_num(sx.float()).to(sx.dtype) if scale == "f32" else sx,
                               laid(clean[1]), sw)
    assert torch.equal(got[~nan], want[~nan])
