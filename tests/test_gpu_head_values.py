"""The class head's rows whose label's logit is not finite, through the label's row of the table alone, on the
GPU. Marked gpu."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import head_oracle as ref  # noqa: E402
from test_gpu_class_loss import DEV, TYPES, inputs, matrix, ops  # noqa: E402,F401


# walks in one part and in several, tiles of few rows and of many, and a single class
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("n, d, v", [(150, 16, 70), (3, 16, 5000), (90, 100, 700), (5, 200, 3000), (150, 200, 70), (40, 16, 1),
                                     (40, 200, 1)])
def test_a_labels_logit_that_is_not_finite(ops, n, d, v, sign, dtype):
    """An infinity in the table's row of row 2's label alone: that row's features are positive there, so its other
    logits are finite."""
    h, w, labels, weights = inputs(n, d, v, 3)
    labels = labels.clamp_min(0)
    h[:, 0] = h[:, 0].abs() + 0.5
    h, w = matrix(h, dtype), matrix(w, dtype)
    hit = int(labels[2])
    w[hit, 0] = sign * float("inf")
    up = weights.abs() + 0.5
    for gradient in ("none", "both"):
        got = ops.class_loss(h, w, labels, row_weights=up, gradient=gradient)
        assert got["loss"][2].isnan() and got["stats"][2, 2].isnan()
        rest = labels != hit
        if sign > 0:  # another class of +inf
            assert got["loss"].isnan().all()
        elif dtype != "f32" and rest.any():  # another class of -inf: none of the probability
            keep = torch.arange(v, device=DEV) != hit
            at = labels - (labels > hit).long()
            want = ref.class_loss(h[rest], w[keep], at[rest], up[rest])["loss"]
            assert ((got["loss"][rest].double() - want).abs() <= 1e-3 * (want.abs() + up[rest])).all()
        if gradient == "both":
            assert got["d_features"][2].isnan().all() and got["d_table"].isnan().all()
    back = ops.class_loss_backward(h, w, labels, got["stats"], up)
    assert back["d_features"][2].isnan().all() and back["d_table"].isnan().all()
    # such a row that does not count stays 0
    up[2] = 0.0
    got = ops.class_loss(h, w, labels, row_weights=up)
    assert got["loss"][2] == 0 and not got["d_features"][2].any()
