"""The class head's cross entropy on the GPU against 64 bits (head_oracle.py).
Marked gpu.

Tolerances, with u = 2^-24. A logit is a sum of D products in fp32: off by at most
D u sum |h W| (A below), fp32 inputs in two fp16 terms by 2^-21 A more (each factor is off by
2^-23 of itself, and the product of the low terms, 2^-22 at most, is left out). The loss
has that twice (the label's logit and the others'), and 60 u of the sums, exponents and logarithm as in
test_gpu_logits.py, its own rounding, and 2 u |x| of the largest exponent. With logits that fp32 holds exactly, only
the latter.

A probability is e^(2 A-term + 3e-5) off (test_gpu_logits.py). d is rounded to 11 bits (2^-11 relative,
below 2^-14 2^-14 2^-25 w / T; 2^-22 for fp32 inputs, whose other factor has 2^-22 too and
whose products of low terms are left out, 2^-22), and sums of K terms are off by K u of the sum of
absolute terms. Results are rounded once: half an ulp of their type."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import head_oracle as ref  # noqa: E402

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"f32": (2.0 ** -24, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from tiny_metal_nn import LogitOps
    with LogitOps() as o:
        yield o


def matrix(values, dtype, pad=0, offset=0):
    """A device matrix with `pad` elements between rows, its data `offset` elements
    into the allocation."""
    n, v = values.shape
    buf = torch.full((offset + n * (v + pad) + 8,), 7.0, device=DEV, dtype=TYPES[dtype])
    z = buf[offset:offset + n * (v + pad)].view(n, v + pad)[:, :v]
    z.copy_(values)
    return z



def inputs(n, d, v, seed, exact=False, lean=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if exact:  # multiples of 1 / 8 up to 2: products of 1 / 64, sums below 2^18 of them
        h = torch.randint(-16, 17, (n, d), device=DEV, generator=g) / 8.0
        w = torch.randint(-16, 17, (v, d), device=DEV, generator=g) / 8.0
        h *= (torch.rand(n, d, device=DEV, generator=g) < 8.0 / max(d, 8)).float()
    else:
        h = torch.randn(n, d, device=DEV, generator=g)
        w = torch.randn(v, d, device=DEV, generator=g) * (1.5 / d ** 0.5)
    labels = torch.randint(0, v, (n,), device=DEV, generator=g)
    if not exact:
        h += lean * w[labels] * torch.rand(n, 1, device=DEV, generator=g)
    if n > 2:
        labels[1] = -1
    weights = torch.randn(n, device=DEV, generator=g)
    if n > 4:
        weights[3] = 0.0
    return h, w, labels, weights


def logit_error(want, d, dtype, t, exact=False):
    """Of each row, relative to 1 in the exponent."""
    if exact:
        return torch.zeros_like(want["loss"])
    return want["z"] / t * (d * U + (2.0 ** -21 if dtype == "f32" else 0.0))


def check_loss(got, want, weights, d, dtype, t, exact=False):
    w = 1.0 if weights is None else weights.double().abs()
    span = want["loss"].abs() + 1
    err = (2 * logit_error(want, d, dtype, t, exact) + 60 * U) * (w + want["loss"].abs()) + 4 * U * w * span
    assert ((got.double() - want["loss"]).abs() <= err + 1e-30).all(), \
        ((got.double() - want["loss"]).abs() / (err + 1e-30)).max()


def check_gradient(got, value, size, prob, terms, floor, dtype):
    """`prob`: the relative error of d; `terms`: of the sum; `floor`: absolute."""
    low = 2.0 ** -11 if dtype != "f32" else 2.0 ** -20
    rel, step = HALF_ULP[dtype]
    err = size * (prob + low + terms * U) + floor
    err = err + rel * (value.abs() + err) + step
    bad = (got.double() - value).abs() > err + 1e-30
    assert not bad.any(), ((got.double() - value).abs() / (err + 1e-30)).max()


def check_all(got, want, h, w, weights, dtype, t, exact=False, names=("d_features", "d_table")):
    n, d = h.shape
    v = w.shape[0]
    up = torch.ones(n, device=DEV, dtype=torch.float64) if weights is None else weights.double().abs()
    if "loss" in got:
        check_loss(got["loss"], want, weights, d, dtype, t, exact)
    prob = 2 * logit_error(want, d, dtype, t, exact).unsqueeze(1) + 3e-5
    least = 2.0 ** -39 / t
    if "d_features" in names:
        floor = least * up.unsqueeze(1) * w.double().abs().sum(0) + 2.0 ** -39 * w.double().abs().max() * want["d"].abs().sum(1, keepdim=True)
        check_gradient(got["d_features"], want["d_features"], want["x"], prob, v, floor, dtype)
    if "d_table" in names:
        most = (up.max() if n else 0.0) * h.double().abs().max()
        floor = least * n * most + 2.0 ** -37 * most * n / t
        check_gradient(got["d_table"], want["d_table"], want["y"], prob.max(), n, floor, dtype)


SHAPES = [(1, 1, 1), (1, 8, 2), (3, 5, 7), (70, 16, 64), (33, 64, 1000), (257, 130, 515), (129, 1000, 131),
          (64, 24, 5003), (300, 300, 300), (1, 520, 4099), (1029, 72, 33), (2, 2050, 3), (40, 128, 2048)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_loss_and_gradients(ops, shape, dtype):
    n, d, v = shape
    rng = np.random.default_rng(n * 31 + d * 7 + v)
    t = float(rng.choice([0.5, 1.0, 2.0]))
    h, w, labels, weights = inputs(n, d, v, n + d + v)
    h = matrix(h, dtype, pad=int(rng.integers(0, 4)), offset=int(rng.integers(0, 3)))
    w = matrix(w, dtype, pad=int(rng.integers(0, 4)), offset=int(rng.integers(0, 3)))
    labels = labels.to(torch.int32 if v % 2 else torch.int64)
    got = ops.class_loss(h, w, labels, temperature=t, row_weights=weights)
    want = ref.class_loss(h, w, labels, weights, t)
    check_all(got, want, h, w, weights, dtype, t)
    # the loss first, its backward pass with the weights; the loss alone
    first = ops.class_loss(h, w, labels, temperature=t, gradient="none")
    assert set(first) == {"loss", "stats"}
    check_loss(first["loss"], ref.class_loss(h, w, labels, None, t), None, d, dtype, t)
    back = ops.class_loss_backward(h, w, labels, first["stats"], weights, temperature=t)
    check_all(back, want, h, w, weights, dtype, t)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(5, 16, 9), (130, 64, 700), (70, 256, 3000)], ids=lambda s: "x".join(map(str, s)))
def test_exact_logits(ops, shape, dtype):
    """Inputs whose logits fp32 holds: the softmax's own errors."""
    n, d, v = shape
    h, w, labels, weights = inputs(n, d, v, 5, exact=True)
    h, w = matrix(h, dtype), matrix(w, dtype)
    got = ops.class_loss(h, w, labels, row_weights=weights)
    check_all(got, ref.class_loss(h, w, labels, weights), h, w, weights, dtype, 1.0, exact=True)


# tiles of 256 x 256 and several pieces of the classes
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(4096, 64, 9000), (8191, 40, 40001), (2048, 512, 8192)],
                         ids=lambda s: "x".join(map(str, s)))
def test_large(ops, shape, dtype):
    n, d, v = shape
    h, w, labels, weights = inputs(n, d, v, 9)
    h, w = matrix(h, dtype), matrix(w, dtype)
    got = ops.class_loss(h, w, labels, row_weights=weights)
    check_all(got, ref.class_loss(h, w, labels, weights), h, w, weights, dtype, 1.0)
