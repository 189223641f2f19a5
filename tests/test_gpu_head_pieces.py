"""Wide calls of the class head that go in several pieces of classes, the last one shorter than the
others by several tiles, against 64 bits. Marked gpu. Tolerances are those of test_gpu_class_loss.py."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import head_oracle as ref  # noqa: E402
from test_gpu_class_loss import TYPES, check_all, inputs, matrix, ops  # noqa: E402,F401


# pieces of 24832 classes, the last one of 24065 (16 bits); of 14336, the last one of 12545 (fp32)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_last_piece_short_by_several_tiles(ops, dtype):
    n, d, v = 4096, 136, 98561
    h, w, labels, weights = inputs(n, d, v, 5)
    labels[:3] = torch.tensor([v - 1, 0, v // 2])
    h, w = matrix(h, dtype), matrix(w, dtype)
    got = ops.class_loss(h, w, labels, row_weights=weights)
    want = ref.class_loss(h, w, labels, weights)
    check_all(got, want, h, w, weights, dtype, 1.0)
    back = ops.class_loss_backward(h, w, labels, got["stats"], weights)
    for name in ("d_features", "d_table"):
        assert torch.equal(back[name], got[name]), name
