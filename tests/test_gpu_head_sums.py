"""The class head's sums over very many classes in one part, on the GPU against 64 bits. Marked gpu."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import head_oracle as ref  # noqa: E402
from test_gpu_class_loss import DEV, TYPES, U, matrix, ops  # noqa: E402,F401


# so many rows that each walks over all classes itself; logits nearly alike, alike but for one class (every term
# of a long sum is rounded, and then in one direction), and rising with the class (a new largest one in every tile)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["near", "alike", "rising"])
@pytest.mark.parametrize("d, v", [(8, 1 << 20), (48, 300001)])
def test_sums_over_very_many_classes(ops, d, v, kind, dtype):
    n = 33000
    g = torch.Generator(device=DEV).manual_seed(7)
    h = matrix(torch.randn(n, d, device=DEV, generator=g), dtype)
    w = torch.randn(v, d, device=DEV, generator=g) * 0.01
    if kind == "alike":
        w[1:] = w[1]
        w[0] = w[1] + 0.1
    elif kind == "rising":
        w = torch.linspace(0, 1, v, device=DEV).unsqueeze(1) * torch.randn(d, device=DEV, generator=g)
    w = matrix(w, dtype)
    labels = torch.randint(0, v, (n,), device=DEV, generator=g)
    got = ops.class_loss(h, w, labels, gradient="none")
    some = torch.arange(0, n, 517, device=DEV)
    want = ref.class_loss(h[some], w, labels[some])
    # 2 A of the logits (d u, fp32 inputs 2^-21 more), 60 u of sums, exponents and logarithm, and 4 u of the loss
    a = 2 * want["z"] * (d * U + (2.0 ** -21 if dtype == "f32" else 0.0))
    err = (a + 60 * U) + 4 * U * (want["loss"] + 1)
    off = (got["loss"][some].double() - want["loss"]).abs()
    assert (off <= err).all(), (off / err).max()
    # the sum itself, relative: over the label's class too, against the largest logit
    total = torch.exp(h[some].double() @ w.double().t() - got["stats"][some, :1].double()).sum(1)
    off = (got["stats"][some, 1].double() / total - 1).abs()
    assert (off <= a + 60 * U).all(), (off / (a + 60 * U)).max()
